"""laya_b200_norm on a GPU against the formula in 64 bits.

Tolerances, from the arithmetic. Statistics and the row are fp32 throughout: a sum of D terms in at
most log2(D) + 32 levels of additions (32 per thread, then a tree) is off by at most (log2 D + 32)
half steps of 2^-24 of the sum of magnitudes, and each element goes through fewer than 10 further
roundings, so y is off by at most 60 * 2^-24 * (|z| / std * |w| + |b|), plus the mean's own error,
which is relative to mean|h|, over std. The output's rounding adds half a step of its type relative
to the value (and the smallest subnormal's half step absolutely).
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import half_step, norm  # noqa: E402

BF, HF, F32, E4 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
FLT_MIN = 2.0 ** -126


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")


def rows_of(g, R, D, dtype, pad=0, scale=1.0, shift=0.0):
    return (scale * torch.randn(R, D + pad, device="cuda", generator=g) + shift).to(dtype)[:, :D]


def formula(x, r, w, b, eps, center):
    """(h, y, bound on |y|'s fp32 error) in 64 bits."""
    h = x.double() + (r.double() if r is not None else 0)
    z = h - h.mean(1, keepdim=True) if center else h
    std = (z.pow(2).mean(1, keepdim=True) + eps).sqrt()
    y = z / std * w.double() + (b.double() if b is not None else 0)
    e = 60 * 2.0 ** -24
    bound = e * ((z / std * w.double()).abs() + (b.double().abs() if b is not None else 0))
    if center:  # the mean's error, and that of h - mean, against mean|h|
        bound = bound + e * (h.abs().mean(1, keepdim=True) + h.abs()) / std * w.double().abs()
    return h, y, bound


def check(x, r, w, b, out, sm, scale, eps, center):
    h, y, bound = formula(x, r, w, b, eps, center)
    if sm is not None:
        t = half_step(sm.dtype)
        assert bool(((sm.double() - h).abs() <= (t + 2.0 ** -23) * h.abs() + 2.0 ** -25).all())
    if out.dtype == E4:
        s = torch.clamp_min(y.abs().amax(1) / 448.0, FLT_MIN)
        slack = bound.amax(1) / 448.0 + 2.0 ** -23 * s
        assert bool(((scale.double() - s).abs() <= slack).all())
        y = y / scale.double()[:, None]
        bound = bound / scale.double()[:, None] + 2.0 ** -22 * y.abs()
        # half a step of e4m3: 2^-4 of the value, and half its smallest subnormal, 2^-10
        bound = bound + 2.0 ** -4 * (y.abs() + bound) + 2.0 ** -10
        assert bool((out.float().abs() <= 448).all())
    else:
        tiny = 2.0 ** -25 if out.dtype == HF else 0.0
        bound = bound + half_step(out.dtype) * (y.abs() + bound) + tiny
    err = (out.double() - y).abs()
    assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("D", [1, 7, 8, 64, 255, 256, 257, 1000, 1024, 1025, 2049, 4096, 5248, 8191, 16384])
@pytest.mark.parametrize("rows", [1, 3, 700])
def test_sizes(D, rows):
    """Every thread layout: one warp, four and sixteen warps a row, one to four pieces a thread."""
    g = torch.Generator(device="cuda").manual_seed(D * 7 + rows)
    x, r = rows_of(g, rows, D, BF), rows_of(g, rows, D, F32, scale=3.0)
    w, b = 1 + 0.1 * torch.randn(D, device="cuda", generator=g), torch.randn(D, device="cuda", generator=g)
    for center in (0, 1):
        out, sm = torch.empty(rows, D, device="cuda", dtype=E4), torch.empty_like(r)
        scale = torch.empty(rows, device="cuda")
        assert norm(x, w, out, resid=r, sum=sm, b=b, scale=scale, center=center) == 0
        check(x, r, w, b, out, sm, scale, 1e-5, center)


@pytest.mark.parametrize("xt", [BF, HF, F32])
@pytest.mark.parametrize("rt", [None, BF, HF, F32])
@pytest.mark.parametrize("ot", [BF, HF, F32, E4])
def test_types(xt, rt, ot):
    g = torch.Generator(device="cuda").manual_seed(3)
    R, D = 37, 768
    x, r = rows_of(g, R, D, xt), None if rt is None else rows_of(g, R, D, rt)
    w = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
    for st in (None, BF, HF, F32):
        sm = None if st is None else torch.empty(R, D, device="cuda", dtype=st)
        out = torch.empty(R, D, device="cuda", dtype=ot)
        scale = torch.empty(R, device="cuda") if ot == E4 else None
        assert norm(x, w, out, resid=r, sum=sm, scale=scale, center=1) == 0
        check(x, r, w, None, out, sm, scale, 1e-5, 1)


@pytest.mark.parametrize("pad", [1, 3, 8, 17])
@pytest.mark.parametrize("D", [5, 129, 1024, 3001, 8191])
@pytest.mark.parametrize("xt,rt", [(HF, BF), (F32, HF), (BF, F32)])
def test_strides_leave_the_padding_alone(pad, D, xt, rt):
    """Padded rows of any alignment: the bytes between rows and behind the last row stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(pad)
    R = 11
    x, r = rows_of(g, R, D, xt, pad), rows_of(g, R, D, rt, pad + 1)
    w = torch.ones(D, device="cuda")
    for ot in (HF, E4, F32):
        store = torch.full((R + 1, D + pad), 7.0, device="cuda").to(ot)
        keep = torch.full((R + 1, D + pad), 5.0, device="cuda")
        scale = torch.empty(R, device="cuda") if ot == E4 else None
        assert norm(x, w, store[:R, :D], resid=r, sum=keep[:R, :D], scale=scale) == 0
        check(x, r, w, None, store[:R, :D], keep[:R, :D], scale, 1e-5, 0)
        assert bool((store[:, D:].float() == 7).all()) and bool((store[R].float() == 7).all())
        assert bool((keep[:, D:] == 5).all()) and bool((keep[R] == 5).all())


def test_misaligned_base():
    g = torch.Generator(device="cuda").manual_seed(1)
    R, D = 5, 512
    x = torch.randn(R * D + 1, device="cuda", generator=g).to(BF)[1:].view(R, D)
    w = torch.randn(D + 1, device="cuda", generator=g)[1:]
    out = torch.empty(R * D + 1, device="cuda", dtype=BF)[1:].view(R, D)
    assert norm(x, w, out) == 0
    check(x, None, w, None, out, None, None, 1e-5, 0)


def test_sum_in_place():
    """The stored sum may be the residual stream or x itself, as a layer updates it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    R, D = 300, 1024
    x, r = rows_of(g, R, D, BF), rows_of(g, R, D, F32)
    w = torch.ones(D, device="cuda")
    out, out2 = (torch.empty(R, D, device="cuda", dtype=BF) for _ in range(2))
    sm, stream_ = torch.empty_like(r), r.clone()
    assert norm(x, w, out, resid=r, sum=sm) == 0
    assert norm(x, w, out2, resid=stream_, sum=stream_) == 0
    assert torch.equal(out, out2) and torch.equal(sm, stream_)
    x2, sm16 = x.clone(), torch.empty_like(x)
    assert norm(x, w, out, resid=r, sum=sm16) == 0
    assert norm(x2, w, out2, resid=r, sum=x2) == 0
    assert torch.equal(out, out2) and torch.equal(sm16, x2)


def test_rows_of_zeros_and_tiny_rows():
    D = 256
    x = torch.zeros(3, D, device="cuda")
    x[1] = 1e-30
    w = torch.full((D,), 1e-10, device="cuda")
    out, scale = torch.empty(3, D, device="cuda", dtype=E4), torch.empty(3, device="cuda")
    assert norm(x, w, out, scale=scale, eps=1e-5) == 0
    assert bool((out.float() == 0).all()) or bool(torch.isfinite(out.float()).all())
    assert scale[0].item() == FLT_MIN and bool((out[0].float() == 0).all())
    assert bool((scale >= FLT_MIN).all())


def test_large_offset_layernorm():
    """A mean far above the spread: the two-pass variance keeps the spread's digits."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = rows_of(g, 64, 1024, F32, shift=3e4)
    w = torch.ones(1024, device="cuda")
    out = torch.empty_like(x)
    assert norm(x, w, out, center=1) == 0
    check(x, None, w, None, out, None, None, 1e-5, 1)


def test_nan_and_infinity_stay_in_their_rows():
    g = torch.Generator(device="cuda").manual_seed(5)
    R, D = 9, 512
    x = rows_of(g, R, D, F32)
    x[3, 100], x[5, 7] = math.nan, math.inf
    w = torch.ones(D, device="cuda")
    out, scale = torch.empty(R, D, device="cuda", dtype=E4), torch.empty(R, device="cuda")
    assert norm(x, w, out, scale=scale) == 0
    good = [i for i in range(R) if i not in (3, 5)]
    check(x[good], None, w, None, out[good], None, scale[good], 1e-5, 0)
    assert math.isnan(scale[3].item()) and bool(out[3].float().isnan().all())
    assert bool(out[5].float().isnan().any())


def test_no_rows():
    w = torch.ones(64, device="cuda")
    out = torch.full((2, 64), 3.0, device="cuda")
    assert norm(out, w, out, rows=0) == 0
    assert bool((out == 3).all())


def test_offsets_past_32_bits():
    """Rows 2^20 elements apart: the last row starts past 2^32 bytes."""
    R, D, step = 2100, 8, 1 << 20
    store = torch.empty(R * step, device="cuda", dtype=BF)
    x = store.view(R, step)[:, :D]
    g = torch.Generator(device="cuda").manual_seed(6)
    x.copy_(torch.randn(R, D, device="cuda", generator=g))
    w = torch.ones(D, device="cuda")
    out = torch.empty(R, D, device="cuda")
    assert norm(x, w, out) == 0
    check(x, None, w, None, out, None, None, 1e-5, 0)


def test_stream_and_graph():
    """On a side stream, and captured and replayed with new inputs."""
    g = torch.Generator(device="cuda").manual_seed(7)
    R, D = 128, 1024
    x, w = rows_of(g, R, D, BF), torch.ones(D, device="cuda")
    out, scale = torch.empty(R, D, device="cuda", dtype=E4), torch.empty(R, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert norm(x, w, out, scale=scale, sync=0) == 0
    torch.cuda.current_stream().wait_stream(s)
    check(x, None, w, None, out, None, scale, 1e-5, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc = norm(x, w, out, scale=scale, sync=0)
        waited = norm(x, w, out, scale=scale, sync=1)
    assert rc == 0 and waited == -2
    x.copy_(rows_of(g, R, D, BF))
    graph.replay()
    torch.cuda.synchronize()
    check(x, None, w, None, out, None, scale, 1e-5, 0)


def test_host_memory_is_refused():
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64)
    out = torch.empty_like(x)
    assert norm(x, w, out) == -2
    assert norm(x, w.cuda(), out.cpu()) == -2
    assert norm(x.cpu().pin_memory(), w.cuda(), out) == -2
