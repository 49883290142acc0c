"""The largest scale and caps that laya_b200_attention_varlen takes, on a GPU."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import attention  # noqa: E402
from tests.test_attention_varlen_gpu import BF, gpu, offsets  # noqa: E402, F401


@pytest.mark.parametrize("lq", [1, 100])
@pytest.mark.parametrize("scale,cap", [(2.0 ** 126, 0.0), (2.0 ** 126, 2.0 ** 126), (1.0, 2.0 ** 126), (2.0 ** -100, 0.0),
                                       (2.0 ** -100, 2.0 ** -100)])
def test_extreme_scales(lq, scale, cap):
    """One key's score is far above the others' (or, with a cap below them, all are alike), while scale, cap or
    their ratio lies near an end of fp32's range."""
    D, n = 64, 200
    q, k = torch.zeros(lq, D, device="cuda", dtype=BF), torch.zeros(n, D, device="cuda", dtype=BF)
    q[:, 0] = min(1.0, 1e30 / scale) if scale > 1 else 2.0 ** 60
    k[:, 0], k[70, 0] = (0.25, 0.5) if scale > 1 else (2.0 ** 45, 2.0 ** 46)
    v = torch.randn(n, D, device="cuda").to(BF)
    out = torch.empty_like(q)
    assert attention(q, k, v, out, None, offsets([lq]), offsets([n]), lq, n, 1, 1, D, scale=scale, cap=cap) == 0
    if cap == 2.0 ** -100:  # every score at the cap: all weights alike
        mean, mag = v.double().mean(0), v.double().abs().mean(0)
        assert bool(((out.double() - mean).abs() <= 2 ** -7 * mag).all())
    else:
        assert torch.equal(out, v[70].expand(lq, D))
