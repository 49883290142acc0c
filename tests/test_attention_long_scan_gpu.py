"""One query of a document that only the last of very many keys belong to: the kernel for few rows skips the
keys before them for longer than any wait inside it may last (about a second), and has to finish all the
same."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.layer_helpers import attention  # noqa: E402
from tests.test_attention_varlen_gpu import BF, check_sequence, gpu, offsets  # noqa: E402, F401


def test_documents_far_apart():
    g = torch.Generator(device="cuda").manual_seed(1)
    n, D = 200_000_000, 64
    kv = torch.zeros(n, D, device="cuda", dtype=BF)  # 25.6 GB, keys and values alike
    dk = torch.full((n,), 3, device="cuda", dtype=torch.int32)
    dk[-10:], dk[:5] = 7, 7
    kv[-100:], kv[:100] = (torch.randn(100, D, device="cuda", generator=g).to(BF) for _ in range(2))
    q = torch.randn(1, D, device="cuda", generator=g).to(BF)
    out, lse = torch.empty_like(q), torch.empty(1, 1, device="cuda")
    rc = attention(q, kv, kv, out, lse, offsets([1]), offsets([n]), 1, n, 1, 1, D,
                   doc_q=torch.tensor([7], device="cuda", dtype=torch.int32), doc_k=dk)
    assert rc == 0
    seen = torch.cat([kv[:5], kv[-10:]]).view(15, 1, D)
    check_sequence(out.view(1, 1, D), lse, q.view(1, 1, D), seen, seen, BF, 0.125)
    del kv, dk, seen
    torch.cuda.empty_cache()
