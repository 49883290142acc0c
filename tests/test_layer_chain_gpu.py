"""The layer operators in the order a layer uses them, on packed sequences: norm to 8 bits, the QKV product
on those 8 bits, masked attention, the output product added to the residual stream, the norm again, and
the MLP's two products, eagerly and replayed from one graph, against the same layer in 64 bits.

Every operator's own error is held by its own tests; here the layer's inputs and outputs are bf16 and
the 8-bit activations carry up to 2^-4 of rounding per element, so the layer is compared with the
64-bit layer that rounds at the same places (to e4m3 with the same scales, to bf16): what is left are
elements at a rounding border that fall the other way. Such an element moves a sum of K terms by at most
2^-3 of one term; the bound below takes 1 % of the elements to do so, at random: an output's relative
error is then at most 2^-3 * sqrt(0.01) of the branch's size for each of the four 8-bit products, 0.05.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import attention, linear, norm  # noqa: E402

BF, E4 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")


def quant(w):
    s = (w.abs().amax(1) / 448).clamp_min(2.0 ** -126)
    return (w / s[:, None]).to(E4), s


def norm8(h, w):
    y = h / (h.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    s = (y.abs().amax(1) / 448).float().double()
    return (y / s[:, None]).float().to(E4).double() * s[:, None]


def test_layer():
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    lens, H, Hkv, D, d, inter = [100, 1, 333, 64], 8, 2, 64, 512, 1536
    T = sum(lens)
    cu = torch.tensor([0, 100, 101, 434, 498], dtype=torch.int32, device="cuda")
    pre = torch.tensor([10, 0, 100, 64], dtype=torch.int32, device="cuda")
    ids = torch.tensor([i // 50 for n in lens for i in range(n)], dtype=torch.int32, device="cuda")
    x0, n1, n2 = 3 * rnd(T, d), 1 + 0.1 * rnd(d), 1 + 0.1 * rnd(d)
    width = (H + 2 * Hkv) * D
    (wq, sq), (wo, so) = quant(rnd(width, d) / math.sqrt(d)), quant(rnd(d, H * D) / math.sqrt(d))
    (wi, si), (wm, sm) = quant(rnd(inter, d) / math.sqrt(d)), quant(rnd(d, inter) / math.sqrt(inter))
    b = 0.1 * rnd(inter)
    x = x0.clone()
    a8, s8 = torch.empty(T, d, device="cuda", dtype=E4), torch.empty(T, device="cuda")
    m8, ms = torch.empty(T, inter, device="cuda", dtype=E4), torch.empty(T, device="cuda")
    qkv, att = torch.empty(T, width, device="cuda", dtype=BF), torch.empty(T, H * D, device="cuda", dtype=BF)
    hid, one = torch.empty(T, inter, device="cuda", dtype=BF), torch.ones(max(d, inter), device="cuda")
    o8, os_ = torch.empty(T, H * D, device="cuda", dtype=E4), torch.empty(T, device="cuda")
    q, k, v = qkv[:, :H * D], qkv[:, H * D:(H + Hkv) * D], qkv[:, (H + Hkv) * D:]

    def layer():
        rc = [norm(x, n1, a8, scale=s8, sync=0),
              linear(a8, wq, qkv, s8, sq, sync=0),
              attention(q, k, v, att, None, cu, cu, max(lens), max(lens), H, Hkv, D, cap=30.0, right=0, prefix=pre,
                        doc_q=ids, doc_k=ids, sync=0),
              norm(att, one[:d], o8, scale=os_, sync=0),
              linear(o8, wo, x, os_, so, resid=x, sync=0),
              norm(x, n2, a8, scale=s8, sync=0),
              linear(a8, wi, hid, s8, si, bias=b, act=2, sync=0),
              norm(hid, one[:inter], m8, scale=ms, sync=0),
              linear(m8, wm, x, ms, sm, resid=x, sync=0)]
        assert rc == [0] * len(rc), rc

    layer()
    torch.cuda.synchronize()
    eager = x.clone()

    f = torch.float64
    W = lambda w, s: w.double() * s.double()[:, None]  # noqa: E731
    h = x0.double()
    z = (norm8(h, n1) @ W(wq, sq).t()).to(BF).double()
    o = torch.zeros(T, H, D, dtype=f, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        r = z[at:at + n]
        qq, kk, vv = (t.reshape(n, -1, D) for t in (r[:, :H * D], r[:, H * D:(H + Hkv) * D], r[:, (H + Hkv) * D:]))
        j = torch.arange(n, device="cuda")
        see = ((j[None] <= j[:, None]) | (j[None] < int(pre[i]))) & (ids[at:at + n, None] == ids[None, at:at + n])
        for e in range(H):
            s = 30 * torch.tanh(qq[:, e] @ kk[:, e // (H // Hkv)].t() / math.sqrt(D) / 30)
            o[at:at + n, e] = torch.softmax(s.masked_fill(~see, -math.inf), 1) @ vv[:, e // (H // Hkv)]
        at += n
    o = o.view(T, H * D).to(BF).double()
    branch1 = norm8(o, torch.ones(H * D, device="cuda")) @ W(wo, so).t()
    h1 = (h + branch1).float().double()
    u = norm8(h1, n2) @ W(wi, si).t() + b.double()
    u = (u * torch.special.ndtr(u)).to(BF).double()
    branch2 = norm8(u, torch.ones(inter, device="cuda")) @ W(wm, sm).t()
    ref = h1 + branch2
    err = (eager.double() - ref).norm() / (branch1.norm() + branch2.norm())
    assert float(err) < 0.05, float(err)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    x.copy_(x0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, eager)


def test_first_call_inside_a_capture_is_refused():
    """In a fresh process: set-up is not done inside a capture (-8), the capture stays usable, and after one
    call outside it the same capture works."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from tests.layer_helpers import norm
x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
out, y = torch.zeros_like(x), torch.zeros_like(x)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y.add_(1)
    rc = norm(x, w, out, sync=0)
assert rc == -8, rc
g.replay()
torch.cuda.synchronize()
assert bool((y == 1).all()) and bool((out == 0).all())
assert norm(x, w, out) == 0
want = out.clone()
out.zero_()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    assert norm(x, w, out, sync=0) == 0
g.replay()
torch.cuda.synchronize()
assert torch.equal(out, want)
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_threads_at_once():
    """Calls from several host threads, each on a stream of its own."""
    import threading
    g = torch.Generator(device="cuda").manual_seed(1)
    A = torch.randn(200, 512, device="cuda", generator=g).to(BF)
    W = torch.randn(300, 512, device="cuda", generator=g).to(BF)
    n = torch.ones(512, device="cuda")
    want, y = torch.empty(200, 300, device="cuda"), torch.empty(200, 512, device="cuda", dtype=BF)
    assert norm(A, n, y) == 0 and linear(y, W, want) == 0
    bad = []

    def work():
        torch.cuda.set_device(0)
        s = torch.cuda.Stream()
        mine, out = torch.empty_like(y), torch.empty_like(want)
        s.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(s):
            for _ in range(50):
                if norm(A, n, mine, sync=0) or linear(mine, W, out, sync=0):
                    bad.append("refused")
        s.synchronize()
        if not torch.equal(out, want):
            bad.append("differs")

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad
    from layamd_b200 import load_lib
    assert load_lib().laya_b200_kernel_error(0) == 0
