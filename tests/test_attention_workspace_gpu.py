"""The workspace query of laya_b200_attention_varlen plans as the call does."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from layamd_b200 import load_lib  # noqa: E402
from tests.layer_helpers import attention  # noqa: E402
from tests.test_attention_varlen_gpu import BF, gpu, offsets  # noqa: E402, F401


@pytest.mark.parametrize("rows,max_k,Hq,Hkv", [(1, 32768, 16, 16), (3, 9000, 8, 2), (100, 9000, 2, 1)])
def test_longest_length_above_the_rows(rows, max_k, Hq, Hkv):
    """A max_q past rows_q changes neither the query's answer nor the call's result."""
    f = load_lib().laya_b200_attention_varlen_ws
    n = f(1, rows, rows, max_k, Hq, Hkv, 64)
    assert n > 0
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(rows, Hq * 64, device="cuda", generator=g).to(BF)
    k, v = (torch.randn(max_k, Hkv * 64, device="cuda", generator=g).to(BF) for _ in range(2))
    got = []
    for mq in (rows, rows + 1, 2048, 1 << 29):
        assert f(1, rows, mq, max_k, Hq, Hkv, 64) == n
        out, lse = torch.empty_like(q), torch.empty(rows, Hq, device="cuda")
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        assert attention(q, k, v, out, lse, offsets([rows]), offsets([max_k]), mq, max_k, Hq, Hkv, 64, ws=ws) == 0
        got.append((out, lse))
    for o, z in got[1:]:
        assert torch.equal(o, got[0][0]) and torch.equal(z, got[0][1])
