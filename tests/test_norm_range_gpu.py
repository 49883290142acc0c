"""laya_b200_norm on rows whose squares, or whose sum, leave fp32's range, beside ordinary rows, which keep their
bits: against the formula in 64 bits with the bounds of the norm's tests."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import norm  # noqa: E402
from tests.test_norm_gpu import BF, E4, F32, check, gpu, rows_of  # noqa: E402, F401

SIZES = [(7, 0), (256, 0), (1024, 0), (1025, 3), (4096, 0), (8191, 1), (16384, 0)]


@pytest.mark.parametrize("D,pad", SIZES)
@pytest.mark.parametrize("center", [0, 1])
@pytest.mark.parametrize("out", [F32, E4])
def test_large_values(D, pad, center, out):
    for xt in (F32, BF):
        g = torch.Generator(device="cuda").manual_seed(D)
        R = 9
        x = rows_of(g, R, D, xt, pad)
        want, keep = torch.empty(R, D, device="cuda", dtype=out), torch.empty(R, device="cuda")
        w = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
        assert norm(x, w, want, scale=keep if out == E4 else None, center=center) == 0
        ordinary = x.clone()
        for row, f in ((1, 1e19), (2, 1e25), (4, 3e37), (7, 1e30)):
            x[row] = (x[row].double() * f).to(xt)
        x[5] = (3e38 * torch.rand(D, device="cuda", generator=g)).to(xt)  # the sum leaves the range too
        got, scale = torch.empty_like(want), torch.empty(R, device="cuda")
        assert norm(x, w, got, scale=scale if out == E4 else None, center=center) == 0
        check(x, None, w, None, got, None, scale if out == E4 else None, 1e-5, center)
        same = [0, 3, 6, 8]
        assert torch.equal(x[same], ordinary[same])
        assert torch.equal(got[same].view(torch.uint8), want[same].view(torch.uint8))


@pytest.mark.parametrize("D,pad", SIZES)
@pytest.mark.parametrize("center", [0, 1])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-33])
def test_tiny_values_with_a_tiny_eps(D, pad, center, eps):
    """(The mean's error is relative to the row's values, down to fp32's subnormal ones.)"""
    g = torch.Generator(device="cuda").manual_seed(D)
    R = 7
    x = rows_of(g, R, D, F32, pad)
    for row, f in ((1, 1e-19), (3, 1e-25), (4, 1e-33)):
        x[row] *= f
    w = torch.ones(D, device="cuda")
    got = torch.empty(R, D, device="cuda")
    assert norm(x, w, got, eps=eps, center=center) == 0
    check(x, None, w, None, got, None, None, eps, center)
    z = torch.zeros(3, D, device="cuda")
    assert norm(z, w, got[:3], eps=eps, center=center) == 0
    assert bool((got[:3] == 0).all()) if eps > 0 else bool(got[:3].isnan().all())


@pytest.mark.parametrize("D", [256, 1025, 8192])
def test_not_finite_rows_beside_large_ones(D):
    g = torch.Generator(device="cuda").manual_seed(D)
    x = rows_of(g, 6, D, F32)
    x[1, 3], x[2, D - 1] = math.nan, math.inf
    x[4] *= 1e30
    got, w = torch.empty(6, D, device="cuda"), torch.ones(D, device="cuda")
    for center in (0, 1):
        assert norm(x, w, got, center=center) == 0
        good = [0, 3, 4, 5]
        check(x[good], None, w, None, got[good], None, None, 1e-5, center)
        assert bool(got[1].isnan().all()) and bool(got[2, D - 1].isnan())
