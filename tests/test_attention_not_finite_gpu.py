"""Queries, keys and values of laya_b200_attention_varlen that are not finite stay with the rows that see them."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import attention  # noqa: E402
from tests.test_attention_varlen_gpu import BF, gpu, offsets  # noqa: E402, F401


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,lq", [(200, 200), (300, 2)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_not_finite(D, n, lq, cap):
    """A NaN in a query spoils its row and head alone; a NaN key the rows that see it (a masked score is
    replaced), an infinite one too unless a cap bounds its score; an infinite value its column of the rows
    that see it."""
    g = torch.Generator(device="cuda").manual_seed(6)
    base = [torch.randn(r, 2 * D, device="cuda", generator=g).to(BF) for r in (lq, n, n)]

    def call(q, k, v, right=0):
        out, lse = torch.empty_like(q), torch.empty(lq, 2, device="cuda")
        assert attention(q, k, v, out, lse, offsets([lq]), offsets([n]), lq, n, 2, 2, D, cap=cap, right=right) == 0
        return out.view(lq, 2, D), lse

    q, k, v = (t.clone() for t in base)
    q[1, D + 5] = math.nan
    out, lse = call(q, k, v)
    bad = torch.zeros(lq, 2, dtype=torch.bool, device="cuda")
    bad[1, 1] = True
    assert bool(out[bad].isnan().all()) and bool(lse[bad].isnan().all())
    assert bool(torch.isfinite(out[~bad].float()).all()) and bool(torch.isfinite(lse[~bad]).all())
    for x in (math.nan, math.inf, -math.inf):
        q, k, v = (t.clone() for t in base)
        k[n - 1, 7], q[:, 7] = x, 1.0  # the causal mask leaves it to the last row
        out, lse = call(q, k, v)
        bad = torch.zeros(lq, 2, dtype=torch.bool, device="cuda")
        bad[lq - 1, 0] = math.isnan(x) or (x > 0 and cap == 0.0)  # (a score of -infinity has weight 0)
        assert bool(out[bad].isnan().all())
        assert bool(torch.isfinite(out[~bad].float()).all()) and bool(torch.isfinite(lse[~bad]).all())
    q, k, v = (t.clone() for t in base)
    v[3, 9] = math.inf
    out, lse = call(q, k, v, right=-1)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[:, 0, 9] = True
    assert not bool(torch.isfinite(out[hit].float()).any()) and bool(torch.isfinite(out[~hit].float()).all())
    assert bool(torch.isfinite(lse).all())
