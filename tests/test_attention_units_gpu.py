"""Batches whose longest sequence says little about the others: sizes of the work plan of
laya_b200_attention_varlen."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import attention  # noqa: E402
from tests.test_attention_varlen_gpu import BF, check_sequence, gpu, offsets, run  # noqa: E402, F401


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("where", [0, 40, 79])
def test_one_long_sequence_among_short_ones(D, where):
    lens = [(7 * i) % 5 * 30 for i in range(80)]
    lens[where] = 3000
    run(lens, D=D, Hq=4, Hkv=2, right=0)
    run(lens, D=D, Hq=2, Hkv=2, left=64, right=64)
    run(lens, [n + 200 for n in lens], D=D, Hq=2, Hkv=1)


@pytest.mark.parametrize("D", [64, 128])
def test_loose_longest_length(D):
    """max_q above every sequence, up to and past the rows."""
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = [(11 * i) % 200 + 1 for i in range(300)]
    T, Hq, Hkv = sum(lens), 4, 2
    q = torch.randn(T, Hq * D, device="cuda", generator=g).to(BF)
    k, v = (torch.randn(T, Hkv * D, device="cuda", generator=g).to(BF) for _ in range(2))
    want, cu = torch.empty_like(q), offsets(lens)
    assert attention(q, k, v, want, None, cu, cu, max(lens), max(lens), Hq, Hkv, D, right=0) == 0
    for mq in (1000, T, 1 << 29):
        out = torch.full_like(q, 7.0)
        assert attention(q, k, v, out, None, cu, cu, mq, max(lens), Hq, Hkv, D, right=0) == 0
        assert torch.equal(out, want)


def test_sequences_that_start_behind_the_first_row_and_shorter_max_q():
    """Rows before the first sequence and behind the last, empty sequences, and a max_q below the longest: what
    is not asked for stays."""
    g = torch.Generator(device="cuda").manual_seed(4)
    D, T = 64, 9000
    q, k, v = (torch.randn(T, D, device="cuda", generator=g).to(BF) for _ in range(3))
    edges = [700] + [700 + 3 * i for i in range(100)] + [6000, 6000, 6100]
    cu = torch.tensor(edges, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    assert attention(q, k, v, out, None, cu, cu, 4000, 6000, 1, 1, D, right=0) == 0
    asked = torch.zeros(T, dtype=torch.bool, device="cuda")
    for a, b in zip(edges, edges[1:]):
        n = min(b - a, 4000)
        if not n:
            continue
        asked[a:a + n] = True
        m = n if b - a <= 4000 else None
        if m:  # (of the longest sequence, 5003 rows, the first 4000: causal rows need only their own keys)
            check_sequence(out[a:b].view(n, 1, D), None, q[a:b].view(n, 1, D), k[a:b].view(n, 1, D), v[a:b].view(n, 1, D),
                           BF, 0.125, right=0)
        else:
            check_sequence(out[a:a + n].view(n, 1, D), None, q[a:a + n].view(n, 1, D), k[a:a + n].view(n, 1, D),
                           v[a:a + n].view(n, 1, D), BF, 0.125, right=0)
    assert bool((out[~asked] == 7).all())


def test_65535_sequences_with_one_long_one():
    """Single tokens under a causal mask, whose output is their own value, and one sequence of 65,536."""
    g = torch.Generator(device="cuda").manual_seed(5)
    B, Hq, D, long_ = 65535, 64, 64, 65536
    lens = [1] * (B - 1)
    lens.insert(1000, long_)
    T = sum(lens)
    cu = torch.tensor(lens, dtype=torch.int64).cumsum(0)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), cu]).to(torch.int32).cuda()
    q = torch.randn(T, Hq * D, device="cuda", generator=g, dtype=torch.bfloat16)
    k, v = (torch.randn(T, D, device="cuda", generator=g, dtype=torch.bfloat16) for _ in range(2))
    out = torch.full_like(q, 7.0)
    assert attention(q, k, v, out, None, cu, cu, long_, long_, Hq, 1, D, left=200, right=0) == 0
    short = torch.ones(T, dtype=torch.bool, device="cuda")
    short[1000:1000 + long_] = False
    assert torch.equal(out[short].view(-1, Hq, D), v[short][:, None].expand(-1, Hq, D))
    for end in (300, 30000, long_):  # windows of the long one
        a, b = 1000 + end - 300, 1000 + end
        check_sequence(out[b - 100:b].view(100, Hq, D)[:, ::9], None, q[b - 100:b].view(100, Hq, D)[:, ::9],
                       k[a:b].view(300, 1, D), v[a:b].view(300, 1, D), BF, 0.125, left=200, right=0)
