"""What a mask hides from a row changes not one bit of it: keys and values after a causal row, outside its
window, or of other documents (finite ones: their values meet a weight of zero)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import attention  # noqa: E402
from tests.test_attention_varlen_gpu import BF, HF, gpu, offsets  # noqa: E402, F401


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq,Hq", [(4, 1), (4, 8), (8, 2), (9, 2), (200, 2)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_later_keys(D, lq, Hq, cap, dtype):
    g = torch.Generator(device="cuda").manual_seed(lq)
    n = 500
    q = torch.randn(lq, Hq * D, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(n, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    cut = n - lq // 2  # rows below lq - lq // 2 see keys below this one at most
    rows = lq - lq // 2
    dq = torch.tensor([0] * rows + [1] * (lq - rows), dtype=torch.int32, device="cuda")
    dk = torch.tensor([0] * cut + [1] * (n - cut), dtype=torch.int32, device="cuda")
    for masks in (dict(right=0), dict(right=0, left=300), dict(doc_q=dq, doc_k=dk)):
        got = []
        for amp in (1.0, 20.0, 0.0):
            k2, v2 = k.clone(), v.clone()
            k2[cut:], v2[cut:] = (amp * k[cut:].float()).to(dtype), (amp * v[cut:].float()).to(dtype)
            out, lse = torch.empty_like(q), torch.empty(lq, Hq, device="cuda")
            assert attention(q, k2, v2, out, lse, offsets([lq]), offsets([n]), lq, n, Hq, 1, D, cap=cap, **masks) == 0
            got.append((out[:rows].clone(), lse[:rows].clone()))
        for o, z in got[1:]:
            assert torch.equal(o, got[0][0]) and torch.equal(z, got[0][1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lq,Hq", [(2, 1), (4, 8), (200, 2)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_keys_of_other_documents_in_between(D, lq, Hq, cap, dtype):
    """Two documents' keys in no order: the scores of one may grow and move its rows' maxima, the other's rows
    stay as they are."""
    g = torch.Generator(device="cuda").manual_seed(lq)
    n = 2000
    q = torch.randn(lq, Hq * D, device="cuda", generator=g).to(dtype)
    k, v = (torch.randn(n, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    dk = (torch.rand(n, device="cuda", generator=g) < 0.5).to(torch.int32)
    dq = (torch.arange(lq, device="cuda") % 2).to(torch.int32)
    mine, theirs = dq == 0, dk == 1
    grow = torch.linspace(1, 60, n, device="cuda")[:, None]
    got = []
    for other in (False, True):
        k2 = torch.where(theirs[:, None] & other, grow * k.float(), k.float()).to(dtype)
        out, lse = torch.empty_like(q), torch.empty(lq, Hq, device="cuda")
        assert attention(q, k2, v, out, lse, offsets([lq]), offsets([n]), lq, n, Hq, 1, D, cap=cap, doc_q=dq, doc_k=dk) == 0
        got.append((out[mine].clone(), lse[mine].clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
