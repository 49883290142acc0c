"""What the values of a laya_b200_attention_varlen call may and may not depend on: nothing outside its
visible keys and its own row, small weights of fp16, caps of any size, values that are not finite."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import attention, half_step  # noqa: E402
from tests.test_attention_varlen_gpu import BF, HF, check_sequence, gpu, offsets  # noqa: E402, F401


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq,lk", [(100, 100), (1, 100), (3, 200), (130, 500)])
@pytest.mark.parametrize("amp", [1.0, 4.0])
def test_capped_rows_do_not_depend_on_what_nobody_sees(D, lq, lk, amp):
    """Rows behind the last sequence, keys behind its end and keys of padding documents may hold anything:
    not one bit of a capped row changes with them."""
    g = torch.Generator(device="cuda").manual_seed(lk)
    tail = 128
    q, k, v = ((amp * torch.randn(n + tail, D, device="cuda", generator=g)).to(HF) for n in (lq, lk, lk))
    dk = torch.zeros(lk + tail, dtype=torch.int32, device="cuda")
    dk[5::7] = -1
    dq = torch.zeros(lq + tail, dtype=torch.int32, device="cuda")
    for docs in (False, True):
        got = []
        for fill in (0.0, 30.0, math.inf, math.nan):
            for t, n in ((q, lq), (k, lk), (v, lk)):
                t[n:] = fill
            if docs:
                k[:lk][dk[:lk] < 0], v[:lk][dk[:lk] < 0] = fill, fill
            out, lse = torch.empty(lq + tail, D, device="cuda", dtype=HF), torch.empty(lq + tail, 1, device="cuda")
            assert attention(q, k, v, out, lse, offsets([lq]), offsets([lk]), lq, lk, 1, 1, D, cap=30.0,
                             doc_q=dq if docs else None, doc_k=dk if docs else None) == 0
            got.append((out[:lq].clone(), lse[:lq].clone()))
        assert bool(torch.isfinite(got[0][1]).all())
        for o, z in got[1:]:
            assert torch.equal(o, got[0][0]) and torch.equal(z, got[0][1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq", [1, 100])
def test_a_capped_row_does_not_depend_on_its_neighbours(D, lq):
    """The first row's scores are small beside the cap; those of the rows after it are not, or are."""
    g = torch.Generator(device="cuda").manual_seed(5)
    n = max(lq, 4)
    q, k, v = (torch.randn(r, D, device="cuda", generator=g).to(HF) for r in (n, 300, 300))
    one = []
    for amp in (1.0, 50.0):
        x = q.clone()
        x[1:] = (amp * q[1:].float()).to(HF)
        out, lse = torch.empty(n, D, device="cuda", dtype=HF), torch.empty(n, 1, device="cuda")
        assert attention(x, k, v, out, lse, offsets([n]), offsets([300]), n, 300, 1, 1, D, cap=30.0) == 0
        one.append((out[0].clone(), lse[0].clone()))
        check_sequence(out.view(n, 1, D), lse, x.view(n, 1, D), k.view(300, 1, D), v.view(300, 1, D), HF, D ** -0.5, 30.0)
    if lq > 4:  # (few rows move their reference maximum together)
        assert torch.equal(one[0][0], one[1][0]) and torch.equal(one[0][1], one[1][1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq", [1, 100])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("high", [1e3, 1e6, 1e7, 1e8, 3e9, 1e15, 1e30])
def test_large_scores(D, lq, dtype, high):
    """Finite scores of any size, of both signs: the largest two keys of a row share it, whatever their
    scores' last places are worth."""
    g = torch.Generator(device="cuda").manual_seed(7)
    n, half = 300, min(high ** 0.5, 3e4) if dtype == HF else high ** 0.5
    scale = high / half ** 2
    for sign in (1.0, -1.0):
        q, k = torch.zeros(lq, D, device="cuda", dtype=dtype), torch.zeros(n, D, device="cuda", dtype=dtype)
        q[:, 3] = sign * half * torch.linspace(0.5, 1, lq, device="cuda")
        k[:, 3] = sign * half * torch.linspace(0.2, 0.6, n, device="cuda")
        k[70, 3], k[130, 3] = sign * half, sign * half
        for other in (1.0, -1.0):  # the largest scores of the row are positive, or all scores negative
            kk = k if other > 0 else -k
            if other < 0:
                kk[70, 3], kk[130, 3] = -sign * half / 8, -sign * half / 8
            v = torch.randn(n, D, device="cuda", generator=g).to(dtype)
            out, lse = torch.empty_like(q), torch.empty(lq, 1, device="cuda")
            assert attention(q, kk, v, out, lse, offsets([lq]), offsets([n]), lq, n, 1, 1, D, scale=scale) == 0
            s = scale * (q[:, 3:4].double() * kk[70, 3].double())
            mean, mag = (v[70] + v[130].float()) / 2, (v[70].float().abs() + v[130].float().abs()) / 2
            assert bool(((out.float() - mean).abs() <= 3 * half_step(dtype) * mag).all())
            assert bool(((lse.double() - (s + math.log(2))).abs() <= 2 ** -21 * (s.abs() + 1)).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq", [1, 100])
@pytest.mark.parametrize("cap,amp", [(1e20, 5e9), (1e30, 1e15), (1e10, 1e5), (1e-20, 1.0)])
def test_caps_of_any_size(D, lq, cap, amp):
    """One key's score is far above the others' (or, with a cap below them, all are alike), whose squares
    leave fp32's range."""
    q, k = torch.zeros(lq, D, device="cuda", dtype=BF), torch.zeros(300, D, device="cuda", dtype=BF)
    q[:, 3], k[:, 3] = amp, amp / 2
    k[70, 3] = 2 * amp
    v = torch.randn(300, D, device="cuda").to(BF)
    out, lse = torch.empty_like(q), torch.empty(lq, 1, device="cuda")
    assert attention(q, k, v, out, lse, offsets([lq]), offsets([300]), lq, 300, 1, 1, D, scale=0.125, cap=cap) == 0
    if cap > 1:
        assert torch.equal(out, v[70].expand(lq, D))
        s = cap * torch.tanh(q[:, 3:4].double() * k[70, 3].double() * 0.125 / cap)
        assert bool(((lse.double() - s).abs() <= 2e-6 * s).all())
    else:
        mean, mag = v.double().mean(0), v.double().abs().mean(0)
        assert bool(((out.double() - mean).abs() <= 2 ** -7 * mag).all())
        assert bool(((lse.double() - math.log(300)).abs() <= 1e-5).all())


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq", [1, 100])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e8])
def test_scores_near_a_large_cap(D, lq, cap):
    """Scores of a tenth to a fifth of a large cap: lse is the largest capped score, which is off by the
    polynomial's error at u = 0.2 (62 / 2835 u^8 = 6e-8 of it) and seven roundings of 2^-24 (u, u^2, four in
    the polynomial's sum that count less than one together, the products with v and log2 e, lse): 5e-7."""
    q, k = torch.zeros(lq, D, device="cuda", dtype=BF), torch.zeros(64, D, device="cuda", dtype=BF)
    q[:, 0] = 1.0
    k[:, 0] = (cap * torch.linspace(0.1, 0.2, 64, device="cuda")).to(BF)
    v = torch.zeros(64, D, device="cuda", dtype=BF)
    out, lse = torch.empty_like(q), torch.empty(lq, 1, device="cuda")
    assert attention(q, k, v, out, lse, offsets([lq]), offsets([64]), lq, 64, 1, 1, D, scale=1.0, cap=cap) == 0
    want = torch.logsumexp(cap * torch.tanh(k[:, 0].double() / cap), 0)
    assert float((lse.double() - want).abs().max()) <= 5e-7 * float(want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq", [1, 100])
def test_many_small_weights_of_fp16_count(D, lq):
    """131,071 keys of weight e^-17.75 = 2^-25.6 each beside one of weight 1: together 0.26 % of the row, each
    below half of fp16's smallest number. A weight may be off by 2^-32 of the largest (half of that number,
    with the weights held 2^7 up), so the output by n 2^-32 and half a step of its own."""
    n = 1 << 17
    q, k = torch.zeros(lq, D, device="cuda", dtype=HF), torch.zeros(n, D, device="cuda", dtype=HF)
    v = torch.ones(n, D, device="cuda", dtype=HF)
    q[:, 0], k[0, 0], v[0] = 4.4375, 4.0, 0.0
    out, lse = torch.empty_like(q), torch.empty(lq, 1, device="cuda")
    assert attention(q, k, v, out, lse, offsets([lq]), offsets([n]), lq, n, 1, 1, D, scale=1.0) == 0
    w = (n - 1) * math.exp(-17.75)
    want = w / (1 + w)
    bound = n * 2.0 ** -32 + (half_step(HF) + 1e-5) * want + 2.0 ** -25
    assert float((out.double() - want).abs().max()) <= bound
    # (a sum of n positive fp32 terms)
    assert float((lse.double() - (17.75 + math.log1p(w))).abs().max()) <= n * 2.0 ** -24 + 17.75 * 2.0 ** -20
