"""laya_b200_linear on a GPU against the formula in 64 bits.

Tolerances, from the arithmetic. Products of 16- and 8-bit values are exact in fp32. A sum of K terms
in fp32 is off by at most K * 2^-23 of the sum of magnitudes in the worst order of additions (a step may
truncate); that worst case is far above what is seen, so the bound used is the smaller of it and
8 * sqrt(K) * 2^-23 of the magnitudes' sum (errors of a sum of independent terms grow with the root
of their number). Scales, bias and residual add fewer than 8 roundings; the activations are off by at
most 1e-6 absolutely (GELU: a published 1.5e-7 bound on erf) plus 8 half steps of the value, and have
slopes of at most 1.13. The output's rounding adds half a step of its type.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import half_step, linear  # noqa: E402

BF, HF, F32, E4 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")


def rows_of(g, R, C, dtype, scale=1.0):
    """Rows that start on 16 bytes; what lies behind column C is NaN."""
    es = 1 if dtype == E4 else 2
    step = (C * es + 15) // 16 * 16 // es
    t = torch.full((R, step), math.nan, device="cuda")
    t[:, :C] = scale * torch.randn(R, C, device="cuda", generator=g)
    return t.to(dtype)[:, :C]


def activation(y, act):
    if act == 1:
        return torch.relu(y)
    if act == 2:
        return y * torch.special.ndtr(y)
    if act == 3:
        return y * torch.sigmoid(y)
    return y


def check(out, A, W, sa, sw, bias, act, resid):
    K = A.shape[1]
    a, w = A.double(), W.double()
    y, mag = a @ w.t(), a.abs() @ w.abs().t()
    if sa is not None:
        y, mag = y * sa.double()[:, None], mag * sa.double().abs()[:, None]
    if sw is not None:
        y, mag = y * sw.double(), mag * sw.double().abs()
    b = bias.double() if bias is not None else torch.zeros(W.shape[0], device="cuda", dtype=torch.double)
    e = mag * min(K, 8 * math.sqrt(K)) * 2.0 ** -23 + 8 * 2.0 ** -24 * (mag + b.abs())
    y = activation(y + b, act)
    e = 1.13 * e + (1e-6 + 8 * 2.0 ** -24 * y.abs() if act else 0)
    if resid is not None:
        y = y + resid.double()
        e = e + 2.0 ** -24 * (y.abs() + e)
    tiny = 2.0 ** -25 if out.dtype == HF else 0.0
    e = e + half_step(out.dtype) * (y.abs() + e) + tiny
    err = (out.double() - y).abs()
    assert bool((err <= e).all()), float((err - e).max())


def case(M, N, K, ab, ot, scales, bias, act, resid, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M * 31 + N * 7 + K)
    A, W = rows_of(g, M, K, ab), rows_of(g, N, K, ab, 1 / math.sqrt(K))
    sa = 0.5 + torch.rand(M, device="cuda", generator=g) if scales else None
    sw = 0.5 + torch.rand(N, device="cuda", generator=g) if scales else None
    b = torch.randn(N, device="cuda", generator=g) if bias else None
    r = torch.randn(M, N, device="cuda", generator=g).to(ot) if resid else None
    out = torch.full((M, N), math.nan, device="cuda", dtype=ot)
    assert linear(A, W, out, sa, sw, b, act, r) == 0
    check(out, A, W, sa, sw, b, act, r)


# every kernel and shape: few rows, one tile per cluster (K cut in 1 to 8, 64 and 128 columns), pairs
SIZES = [(1, 8, 16), (1, 5248, 1024), (3, 1, 1), (7, 33, 100), (16, 1024, 2624), (16, 9601, 72), (17, 64, 64),
         (17, 1, 5), (33, 100, 1000), (77, 1153, 999), (128, 128, 128), (129, 129, 129), (200, 1024, 1024),
         (512, 1024, 2624), (300, 1000, 64), (1000, 1000, 300), (1023, 2047, 515), (2048, 2304, 768),
         (4099, 1025, 1000), (3000, 5248, 1024), (40, 16384, 200), (5000, 40, 640),
         # a weight so large that the tile kernel takes a few rows too
         (1, 16390, 6200), (9, 13000, 8200)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("ab", [BF, HF, E4])
def test_sizes(M, N, K, ab):
    case(M, N, K, ab, BF, scales=ab == E4, bias=True, act=0, resid=False)


@pytest.mark.parametrize("M,N,K", [(5, 1000, 300), (100, 1000, 600), (600, 640, 1000), (2600, 2311, 200)])
@pytest.mark.parametrize("ab", [BF, HF, E4])
@pytest.mark.parametrize("ot", [BF, HF, F32])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
def test_epilogues(M, N, K, ab, ot, act):
    case(M, N, K, ab, ot, scales=False, bias=False, act=act, resid=False)
    case(M, N, K, ab, ot, scales=True, bias=True, act=act, resid=True, seed=1)


@pytest.mark.parametrize("M,N,K", [(4, 77, 64), (70, 77, 128), (2100, 2100, 64)])
@pytest.mark.parametrize("pad", [1, 3, 8])
@pytest.mark.parametrize("ot", [HF, F32])
def test_strided_output_in_place(M, N, K, pad, ot):
    """The residual stream updated in place in padded storage: nothing outside its columns changes."""
    g = torch.Generator(device="cuda").manual_seed(pad)
    A, W = rows_of(g, M, K, HF), rows_of(g, N, K, HF, 0.1)
    store = torch.randn(M + 1, N + pad, device="cuda", generator=g).to(ot)
    before = store.clone()
    x = store[:M, :N]
    assert linear(A, W, x, resid=x) == 0
    check(x, A, W, None, None, None, 0, before[:M, :N])
    assert torch.equal(store[:, N:], before[:, N:]) and torch.equal(store[M], before[M])


def test_misaligned_output():
    g = torch.Generator(device="cuda").manual_seed(3)
    for M in (2, 300, 2600):
        A, W = rows_of(g, M, 64, BF), rows_of(g, 2600, 64, BF)
        out = torch.empty(M * 2600 + 1, device="cuda", dtype=BF)[1:].view(M, 2600)
        assert linear(A, W, out) == 0
        check(out, A, W, None, None, None, 0, None)


def test_fused_rows_of_a_wider_matrix():
    """A and W as column ranges of wider rows (strides above K)."""
    g = torch.Generator(device="cuda").manual_seed(4)
    for M in (1, 9, 130, 2600):
        wide, wide_w = rows_of(g, M, 640, BF), rows_of(g, 2600, 512, BF, 0.1)
        A, W = wide[:, 64:64 + 200], wide_w[:, 8:208]
        out = torch.empty(M, 2600, device="cuda", dtype=BF)
        assert linear(A, W, out) == 0
        check(out, A, W, None, None, None, 0, None)


def test_e4m3_extremes_are_exact():
    """The largest and smallest 8-bit values: every product and these short sums are exact."""
    vals = torch.tensor([448.0, -448.0, 2.0 ** -9, 0.0, 1.0, -2.0 ** -6, 240.0, 0.875], device="cuda")
    for M, N in ((3, 40), (100, 200), (2600, 2600)):
        A = vals[torch.arange(M * 16, device="cuda") % 8].view(M, 16).to(E4)
        W = vals[(torch.arange(N * 16, device="cuda") // 3) % 8].view(N, 16).to(E4)
        out = torch.empty(M, N, device="cuda")
        assert linear(A, W, out) == 0
        ref = A.double() @ W.double().t()
        mag = A.double().abs() @ W.double().abs().t()
        assert bool(((out.double() - ref).abs() <= 16 * 2.0 ** -23 * mag).all())


def test_nan_rows_and_columns_stay_apart():
    g = torch.Generator(device="cuda").manual_seed(5)
    for M, N in ((5, 100), (140, 300), (2600, 2600)):
        A, W = rows_of(g, M, 96, BF), rows_of(g, N, 96, BF)
        A[M - 2, 5], W[7, 95] = math.nan, math.inf
        out = torch.empty(M, N, device="cuda")
        assert linear(A, W, out, act=1) == 0
        bad = torch.zeros(M, N, device="cuda", dtype=torch.bool)
        bad[M - 2] = True
        assert bool(out[M - 2].isnan().all())
        bad[:, 7] = True
        assert bool(torch.isfinite(out[~bad]).all())


@pytest.mark.parametrize("M,N,K", [(4, 1000, 4096), (100, 512, 4096), (3000, 2304, 512)])
def test_runs_are_bitwise_equal_and_capture(M, N, K):
    """The same bits in every run, on a side stream and replayed from a graph with new inputs."""
    g = torch.Generator(device="cuda").manual_seed(6)
    A, W = rows_of(g, M, K, HF), rows_of(g, N, K, HF)
    out, again, third = (torch.empty(M, N, device="cuda") for _ in range(3))
    assert linear(A, W, out) == 0
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            assert linear(A, W, again, sync=0) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc = linear(A, W, third, sync=0)
    assert rc == 0
    A.copy_(rows_of(g, M, K, HF))
    graph.replay()
    torch.cuda.synchronize()
    assert linear(A, W, out) == 0
    assert torch.equal(out, third)


def test_two_streams_at_once():
    g = torch.Generator(device="cuda").manual_seed(7)
    shapes = [(100, 512, 4096), (2600, 2600, 256), (6, 3000, 2048)]
    ins = [(rows_of(g, m, k, BF), rows_of(g, n, k, BF)) for m, n, k in shapes]
    want = [torch.empty(m, n, device="cuda") for m, n, _ in shapes]
    got = [torch.empty(m, n, device="cuda") for m, n, _ in shapes]
    for (a, w), o in zip(ins, want):
        assert linear(a, w, o) == 0
    streams = [torch.cuda.Stream() for _ in shapes]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (a, w), o in zip(streams, ins, got):
            with torch.cuda.stream(s):
                assert linear(a, w, o, sync=0) == 0
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_empty():
    A = torch.ones(4, 16, device="cuda", dtype=BF)
    out = torch.full((4, 4), 3.0, device="cuda")
    assert linear(A, A, out, M=0) == 0 and linear(A, A, out, N=0) == 0
    assert bool((out == 3).all())


def test_offsets_past_32_bits():
    """A, out and resid rows spread over more than 2^32 bytes."""
    g = torch.Generator(device="cuda").manual_seed(8)
    M, N, K, step = 2200, 16, 32, 1 << 20
    big = torch.empty(M * step, device="cuda", dtype=BF)
    A = big.view(M, step)[:, :K]
    A.copy_(torch.randn(M, K, device="cuda", generator=g))
    out = big.view(M, step)[:, 4096:4096 + N]
    W = rows_of(g, N, K, BF)
    assert linear(A, W, out) == 0
    check(out, A, W, None, None, None, 0, None)
