"""laya_b200_norm with its sum stored over x or resid, at alignments where neighbouring threads and warps read
and write 16-byte pieces of one another's elements: the same bits as with a sum of its own."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import norm  # noqa: E402
from tests.test_norm_gpu import BF, E4, F32, HF, gpu, rows_of  # noqa: E402, F401


@pytest.mark.parametrize("D", [5, 129, 255, 1025, 3001, 5249, 8191, 16383, 16384])
@pytest.mark.parametrize("pad", [0, 1, 3, 8])
@pytest.mark.parametrize("xt,rt", [(HF, BF), (BF, F32), (F32, HF), (F32, F32)])
def test_sum_over_an_input(D, pad, xt, rt):
    g = torch.Generator(device="cuda").manual_seed(D + pad)
    R = 37
    x, r = rows_of(g, R, D, xt, pad), rows_of(g, R, D, rt, pad + 1)
    w = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
    for over in ("x", "resid"):
        src = x if over == "x" else r
        want, own = torch.empty(R, D, device="cuda", dtype=E4), torch.empty_strided(src.shape, src.stride(), dtype=src.dtype,
                                                                                    device="cuda")
        s0, s1 = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
        assert norm(x, w, want, resid=r, sum=own, scale=s0, center=1) == 0
        for _ in range(5):
            store = src._base.clone() if src._base is not None else src.clone()
            over_it = store.as_strided(src.shape, src.stride())
            got = torch.empty_like(want)
            assert norm(over_it if over == "x" else x, w, got, resid=over_it if over == "resid" else r, sum=over_it,
                        scale=s1, center=1) == 0
            assert torch.equal(over_it, own) and torch.equal(s0, s1)
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))
            if pad or over == "resid":  # the padding stays
                base = src._base if src._base is not None else src
                assert torch.equal(store[:, D:], base[:, D:])
