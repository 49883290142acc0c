"""laya_b200_attention_varlen on a GPU against the formula in 64 bits, sequence by sequence.

Tolerances, from the arithmetic. A score is a sum of D exact products in fp32: off by at most D * 2^-23
of the sum of magnitudes (a step may truncate), then scaled, capped (at most 1e-6 of the cap) and biased
with fewer than 8 roundings of 2^-24 of its size; call the largest such error of a row's scores d. The
weights p are rounded to the 16-bit type for the product with v but not in their sum, so an output is off
by at most (u + 2 d + 2^-20) sum_j w_j |v_j| with u half a step of the type, for fp16 also half its
smallest subnormal per key against a row sum of at least 1, and half a step of the output itself. lse
is off by d, by the rounding of a sum of n positive fp32 terms (n * 2^-24) and by 2^-21 of its size.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from layamd_b200 import load_lib  # noqa: E402
from tests.layer_helpers import attention, half_step  # noqa: E402

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")


def offsets(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")


def check_sequence(o, lse, q, k, v, dtype, scale, cap=0.0, slopes=None, left=-1, right=-1, prefix=0, dq=None, dk=None):
    """o [n][Hq][D], lse [n][Hq] of one sequence against q [n][Hq][D], k, v [m][Hkv][D]."""
    n, Hq, D = q.shape
    m, Hkv = k.shape[:2]
    if n == 0:
        return
    G = Hq // Hkv
    pos = torch.arange(n, device="cuda")[:, None] + m - n
    key = torch.arange(m, device="cuda")[None]
    see = torch.ones(n, m, dtype=torch.bool, device="cuda")
    if left >= 0:
        see &= key >= pos - left
    if right >= 0:
        see &= key <= pos + right
    see |= key < prefix
    if dq is not None:
        see &= (dq[:, None] == dk[None]) & (dk >= 0)[None]
    for h in range(Hq):
        qh = q[:, h].double()
        if m == 0:
            assert bool((o[:, h] == 0).all()) and (lse is None or bool((lse[:, h] == -math.inf).all()))
            continue
        # keys that nobody sees may hold anything
        dead = ~see.any(0)
        kh = torch.where(dead[:, None], 0.0, k[:, h // G].double())
        vh = torch.where(dead[:, None], 0.0, v[:, h // G].double())
        s = scale * (qh @ kh.t())
        d = D * 2.0 ** -23 * scale * (qh.abs() @ kh.abs().t())
        if cap > 0:
            s = cap * torch.tanh(s / cap)
            d = d + 1e-6 * cap
        if slopes is not None:
            bias = slopes[h].double() * (pos - key).abs()
            s = s - bias
            d = d + 2.0 ** -22 * bias
        d = torch.where(see, d + 2.0 ** -21 * s.abs(), 0.0).amax(1)
        s = s.masked_fill(~see, -math.inf)
        z = torch.logsumexp(s, 1)
        w = torch.where(see, torch.exp(s - torch.where(z == -math.inf, 0.0, z)[:, None]), 0.0)
        ref, mag = w @ vh, w @ vh.abs()
        u = half_step(dtype)
        e = (u + 2 * d[:, None] + 2.0 ** -20) * mag
        if dtype == HF:
            e = e + 2.0 ** -25 * m * vh.abs().amax() + 2.0 ** -25
        e = e + u * (ref.abs() + e)
        err = (o[:, h].double() - ref).abs()
        assert bool((err <= e).all()), (h, float((err - e).max()), float(err.max()))
        if lse is not None:
            got = lse[:, h].double()
            empty = z == -math.inf
            assert bool((got[empty] == -math.inf).all())
            le = (got - z).abs()[~empty]
            lb = (d + (m + 64) * 2.0 ** -24 + 2.0 ** -21 * (z.abs() + 1))[~empty]
            assert bool((le <= lb).all()), (h, float((le - lb).max()))


def run(lq, lk=None, Hq=4, Hkv=4, D=64, dtype=BF, seed=0, cap=0.0, slopes=False, left=-1, right=-1, prefix=None,
        docs=None, scale=None, fused=False, tail=3, ws="full", amp=1.0, garbage=True, grow=False):
    """One call and its check. docs: (doc_q, doc_k) lists per sequence. Rows behind the last sequence hold NaN
    in k and v, and a mark in out that has to stay."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    lk = lq if lk is None else lk
    Tq, Tk = sum(lq), sum(lk)
    rnd = lambda r, c: (amp * torch.randn(r, c, device="cuda", generator=g)).to(dtype)  # noqa: E731
    if fused:
        x = rnd(Tq + tail, (Hq + 2 * Hkv) * D)
        q, k, v = x[:, :Hq * D], x[:, Hq * D:(Hq + Hkv) * D], x[:, (Hq + Hkv) * D:]
    else:
        q, k, v = rnd(Tq + tail, Hq * D), rnd(Tk + tail, Hkv * D), rnd(Tk + tail, Hkv * D)
    if grow:  # every chunk of keys raises the rows' maximum by far more than the kernels' threshold
        at = 0
        for n in lk:
            k[at:at + n] = k[at:at + n].abs() * torch.linspace(0.1, 12, max(n, 1), device="cuda")[:n, None].to(dtype)
            at += n
        q.copy_(q.abs())
    if garbage and tail:
        k[Tk:], v[Tk:] = math.nan, math.inf
    out = torch.full((Tq + tail, Hq * D), 7.0, device="cuda", dtype=dtype)
    lse = torch.full((Tq + tail, Hq), 7.0, device="cuda")
    cq, ck = offsets(lq), offsets(lk)
    sl = torch.tensor([0.02 * (h + 1) for h in range(Hq)], device="cuda") if slopes else None
    pre = None if prefix is None else torch.tensor(prefix, dtype=torch.int32, device="cuda")
    dq = dk = None
    if docs is not None:
        pad = [0] * tail
        dq = torch.tensor(sum(docs[0], []) + pad, dtype=torch.int32, device="cuda")
        dk = torch.tensor(sum(docs[1], []) + pad, dtype=torch.int32, device="cuda")
        dead = torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
        dead[:Tk] = dk[:Tk] < 0
        k[dead], v[dead] = math.inf, math.nan  # padding documents hold anything
    mq, mk = max(lq), max(lk)
    n = load_lib().laya_b200_attention_varlen_ws(len(lq), Tq + tail, mq, mk, Hq, Hkv, D)
    assert n >= 0
    w = torch.full((n,), 255, dtype=torch.uint8, device="cuda") if n and ws == "full" else None
    sc = D ** -0.5 if scale is None else scale
    rc = attention(q, k, v, out, lse, cq, ck, mq, mk, Hq, Hkv, D, sc, cap, sl, left, right, pre, dq, dk, w)
    assert rc == 0, rc
    a = b = 0
    for i, (x, y) in enumerate(zip(lq, lk)):
        check_sequence(out[a:a + x].view(x, Hq, D), lse[a:a + x], q[a:a + x].reshape(x, Hq, D),
                       k[b:b + y].reshape(y, Hkv, D), v[b:b + y].reshape(y, Hkv, D), dtype, sc, cap, sl, left, right,
                       0 if prefix is None else min(max(prefix[i], 0), y), None if dq is None else dq[a:a + x],
                       None if dk is None else dk[b:b + y])
        a, b = a + x, b + y
    assert bool((out[Tq:] == 7).all()) and bool((lse[Tq:] == 7).all())
    return out, lse


RAGGED = [1, 17, 63, 64, 65, 127, 128, 129, 0, 300, 513]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("fused", [False, True])
def test_ragged(D, dtype, fused):
    run(RAGGED, D=D, dtype=dtype, fused=fused)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("left,right", [(-1, 0), (0, 0), (64, 64), (5, -1), (-1, 7), (100, 0), (0, 200)])
def test_windows(D, left, right):
    run(RAGGED, D=D, left=left, right=right, Hq=4, Hkv=2)
    run([1, 5, 130, 70, 0], [300, 2, 130, 1000, 40], D=D, left=left, right=right)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap,slopes", [(0.0, True), (2.0, False), (30.0, False), (20.0, True)])
def test_caps_and_slopes(D, cap, slopes):
    """Small scores and, with amp 4, scores far beyond the cap."""
    for amp in (1.0, 4.0):
        run([70, 257, 400], D=D, cap=cap, slopes=slopes, amp=amp, right=0)
        run([3, 1, 2], [500, 7, 1300], D=D, cap=cap, slopes=slopes, amp=amp, Hq=4, Hkv=1)


@pytest.mark.parametrize("D", [64, 128])
def test_tiny_cap(D):
    """A cap far below the scores (every score at +-cap, all weights nearly alike), and rows of zero scores."""
    run([200, 70], D=D, cap=1e-7)
    run([1, 2], [300, 90], D=D, cap=1e-7)
    run([200], D=D, cap=1e-7, amp=0.0)


@pytest.mark.parametrize("D", [64, 128])
def test_prefixes(D):
    """Prefixes of no, some and all keys, with windows that leave a gap behind them, and out of range."""
    lens = [200, 513, 700, 64, 1]
    for left, right in ((-1, 0), (40, 0), (10, 10)):
        run(lens, D=D, left=left, right=right, prefix=[0, 100, 129, 64, 1])
        run(lens, D=D, left=left, right=right, prefix=[-5, 10000, 7, 63, 0])
        run([1, 3, 2], [900, 700, 2], D=D, left=left, right=right, prefix=[100, 0, 1], Hq=4, Hkv=2)


def doc_list(rng, n, mean):
    ids, d = [], 0
    while len(ids) < n:
        ids += [-1 if rng.random() < 0.15 else d] * min(n - len(ids), 1 + int(rng.random() * 2 * mean))
        d += 1
    return ids


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mean", [3, 40, 500])
def test_documents(D, mean):
    """Runs of documents with padding between them; also ids in no order and queries of unknown documents."""
    import random
    rng = random.Random(mean)
    lens = [1, 64, 200, 513, 1000]
    ids = [doc_list(rng, n, mean) for n in lens]
    run(lens, D=D, docs=(ids, ids))
    run(lens, D=D, docs=(ids, ids), right=0, left=300, Hq=4, Hkv=2, cap=20.0)
    run(lens, D=D, docs=(ids, ids), right=0, prefix=[1, 10, 100, 300, 64])
    mixed = [[rng.choice([-1, 0, 1, 2, 1 << 30]) for _ in range(n)] for n in lens]
    other = [[rng.choice([-7, 0, 1, 5]) for _ in range(n)] for n in lens]
    run(lens, D=D, docs=(other, mixed))
    lq, lk = [1, 2, 1, 0], [2000, 300, 5, 9]
    kd = [doc_list(rng, n, mean) for n in lk]
    run(lq, lk, D=D, docs=([x[len(x) - n:] for x, n in zip(kd, lq)], kd), Hq=8, Hkv=2)


def test_whole_sequences_of_padding():
    ids = [[-1] * 100, [0] * 50 + [-1] * 150, [-1] * 3]
    for D in (64, 128):
        out, lse = run([100, 200, 3], D=D, docs=(ids, ids))
        assert bool((out[:100] == 0).all()) and bool((lse[:100] == -math.inf).all())
        run([1, 1, 1], [100, 200, 3], D=D, docs=([[0]] * 3, ids))


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (2, 1), (6, 2), (8, 1), (12, 4), (24, 3), (64, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_shared_heads(Hq, Hkv, D):
    run([40, 200], D=D, Hq=Hq, Hkv=Hkv, right=0)
    run([1, 2, 1, 1], [1, 17, 300, 2049], D=D, Hq=Hq, Hkv=Hkv, right=0)


@pytest.mark.parametrize("lq", [1, 2, 4, 5, 16, 17, 33])
@pytest.mark.parametrize("lk", [1, 15, 16, 127, 129, 1000, 5000])
def test_few_queries(lq, lk):
    """Around the border between the two kernels, with queries that lie before the first key (lq > lk)."""
    run([lq, 1], [lk, 3], D=128, Hq=4, Hkv=1, right=0)
    run([lq], [lk], D=64, Hq=2, Hkv=2, right=0, ws="none")
    run([lq], [lk], D=64, Hq=2, Hkv=2, left=50, right=2, dtype=HF)


@pytest.mark.parametrize("D", [64, 128])
def test_more_queries_than_keys(D):
    """Rows before the first key see nothing under a causal mask."""
    out, lse = run([300, 100], [10, 0], D=D, right=0)
    assert bool((out[:290] == 0).all()) and bool((lse[:290] == -math.inf).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_growing_scores(D, dtype):
    run([700, 300], D=D, dtype=dtype, grow=True, scale=0.05)
    run([700, 300], D=D, dtype=dtype, grow=True, scale=0.05, cap=40.0)
    run([1, 2], [3000, 500], D=D, dtype=dtype, grow=True, scale=0.05)


@pytest.mark.parametrize("lq,Hq,Hkv", [(1, 2, 2), (3, 8, 2), (100, 2, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_split_keys_join(lq, Hq, Hkv, D):
    """Few rows over many keys: key ranges and their join, against the call without a workspace, with
    parts that see nothing (documents, window)."""
    lk = 9000
    n = load_lib().laya_b200_attention_varlen_ws(1, lq + 3, lq, lk, Hq, Hkv, D)
    assert n > 0
    run([lq], [lk], D=D, Hq=Hq, Hkv=Hkv)
    run([lq], [lk], D=D, Hq=Hq, Hkv=Hkv, ws="none")
    run([lq], [lk], D=D, Hq=Hq, Hkv=Hkv, right=0, left=700, prefix=[90])
    kd = [[i // 1500 for i in range(lk)]]
    run([lq], [lk], D=D, Hq=Hq, Hkv=Hkv, docs=([[5] * (lq - 1) + [9]], kd))


def test_long_keys_and_many_chunks_of_documents():
    """More chunks than the kernel's document map holds (4096 chunks of 64 keys)."""
    lk = 4096 * 64 + 1000
    kd = [[i // 20000 for i in range(lk)]]
    run([70], [lk], D=64, Hq=1, Hkv=1, docs=([[12] * 30 + [13] * 30 + [3] * 10], kd))


def test_bad_offsets_stay_inside():
    """Offsets outside the arrays or running backwards are cut; nothing outside the rows is written."""
    g = torch.Generator(device="cuda").manual_seed(1)
    Hq = Hkv = 2
    D, T = 64, 100
    q, k, v = (torch.randn(T, Hq * D, device="cuda", generator=g).to(BF) for _ in range(3))
    for cu in ([0, 50, 1 << 30], [-9, 20, 10], [90, 5, 120], [2 ** 31 - 1, -2 ** 31, 7]):
        c = torch.tensor(cu, dtype=torch.int32, device="cuda")
        for mq in (1, T):
            out = torch.zeros(T, Hq * D, device="cuda", dtype=BF)
            assert attention(q, k, v, out, None, c, c, mq, T, Hq, Hkv, D) == 0
            assert bool(torch.isfinite(out.float()).all())


def test_shorter_max_q_leaves_later_rows():
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(300, 128, device="cuda", generator=g).to(BF) for _ in range(3))
    c = offsets([300])
    for mq in (130, 8):
        out = torch.full((300, 128), 7.0, device="cuda", dtype=BF)
        assert attention(q, k, v, out, None, c, c, mq, 300, 2, 2, 64) == 0
        assert bool((out[mq:] == 7).all())
        check_sequence(out[:mq].view(mq, 2, 64), None, q.view(300, 2, 64)[:mq], k.view(300, 2, 64), v.view(300, 2, 64),
                       BF, 0.125)


def test_nothing_to_do():
    q = torch.randn(4, 64, device="cuda").to(BF)
    out = torch.full_like(q, 7.0)
    c = offsets([4])
    assert attention(q, q, q, out, None, c, c, 0, 4, 1, 1, 64) == 0
    assert attention(q[:0], q, q, out[:0], None, c, c, 4, 4, 1, 1, 64) == 0
    assert bool((out == 7).all())
    none = torch.empty(0, 64, device="cuda", dtype=BF)
    for mq in (1, 4):
        assert attention(q, none, none, out, None, c, offsets([0]), mq, 0, 1, 1, 64) == 0
    torch.cuda.synchronize()
    assert bool((out == 0).all())
    many = torch.randn(200, 64, device="cuda").to(BF)
    out = torch.full_like(many, 7.0)
    assert attention(many, none, none, out, None, offsets([200]), offsets([0]), 200, 0, 1, 1, 64) == 0
    torch.cuda.synchronize()
    assert bool((out == 0).all())


@pytest.mark.parametrize("lq,lk", [([300, 77], None), ([1, 1], [5000, 3000])])
def test_bitwise_stable_on_streams_and_in_graphs(lq, lk):
    g = torch.Generator(device="cuda").manual_seed(3)
    lk = lq if lk is None else lk
    Hq, Hkv, D = 8, 2, 128
    q = torch.randn(sum(lq), Hq * D, device="cuda", generator=g).to(BF)
    k, v = (torch.randn(sum(lk), Hkv * D, device="cuda", generator=g).to(BF) for _ in range(2))
    cq, ck = offsets(lq), offsets(lk)
    n = load_lib().laya_b200_attention_varlen_ws(len(lq), q.shape[0], max(lq), max(lk), Hq, Hkv, D)
    sets = []
    for _ in range(3):
        sets.append((torch.empty_like(q), torch.empty(q.shape[0], Hq, device="cuda"),
                     torch.empty(n, dtype=torch.uint8, device="cuda") if n else None))
    call = lambda s, sync: attention(q, k, v, s[0], s[1], cq, ck, max(lq), max(lk), Hq, Hkv, D, cap=30.0, right=0,  # noqa: E731
                                     ws=s[2], sync=sync)
    assert call(sets[0], 1) == 0
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for st, s in zip(streams, sets[1:]):
            with torch.cuda.stream(st):
                assert call(s, 0) == 0
    torch.cuda.synchronize()
    for s in sets[1:]:
        assert torch.equal(s[0], sets[0][0]) and torch.equal(s[1], sets[0][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc = call(sets[1], 0)
    assert rc == 0
    q.copy_(torch.randn(q.shape, device="cuda", generator=g))
    graph.replay()
    torch.cuda.synchronize()
    assert call(sets[0], 1) == 0
    assert torch.equal(sets[1][0], sets[0][0]) and torch.equal(sets[1][1], sets[0][1])


def test_key_offsets_past_32_bits():
    """A cache whose rows lie far apart: the last key starts past 2^32 bytes."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n, D, step = 2300, 64, 1 << 20
    big = torch.empty(n * step, device="cuda", dtype=BF).view(n, step)
    k, v = big[:, :D], big[:, 4096:4096 + D]
    k.copy_(torch.randn(n, D, device="cuda", generator=g))
    v.copy_(torch.randn(n, D, device="cuda", generator=g))
    for lq in (1, 200):
        q = torch.randn(lq, D, device="cuda", generator=g).to(BF)
        out = torch.empty_like(q)
        assert attention(q, k, v, out, None, offsets([lq]), offsets([n]), lq, n, 1, 1, D) == 0
        check_sequence(out.view(lq, 1, D), None, q.view(lq, 1, D), k.reshape(n, 1, D), v.reshape(n, 1, D), BF, 0.125)


@pytest.mark.parametrize("D", [64, 128])
def test_many_tiles_that_see_nothing_between_others(D):
    """More units than the GPU runs at once, most of them without a visible key: runs of such units
    between ordinary ones, in every order that a CTA meets them."""
    import random
    rng = random.Random(5)
    lens = [rng.choice([128, 200, 300]) for _ in range(260)]
    ids = [[-1 if i % 7 else 0] * n for i, n in enumerate(lens)]
    out, lse = run(lens, D=D, Hq=4, Hkv=2, docs=(ids, ids))
    assert bool((lse[:lens[0]] > -math.inf).all()) and bool((lse[lens[0]:lens[0] + lens[1]] == -math.inf).all())
