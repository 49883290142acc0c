"""One row has no stride of its own: the layer operators take any stride with it, on a GPU and (the checks of
arguments alone) without one."""
import pytest

torch = pytest.importorskip("torch")

from tests.layer_helpers import attention, linear  # noqa: E402
from tests.test_layer_refusals_cpu import L, attn_args, linear_args  # noqa: E402, F401

STRIDES = [0, 1, 8, 63, 64, 65, 999, 1 << 33, -5]


@pytest.mark.parametrize("ld", STRIDES)
def test_accepted(L, ld):  # noqa: F811
    assert L.laya_b200_linear(*linear_args(M=1, lda=ld, ldo=ld, ldr=ld)) == -1
    assert L.laya_b200_linear(*linear_args(N=1, ldw=ld)) == -1
    f = L.laya_b200_attention_varlen
    assert f(*attn_args(rows_q=1, ldq=ld, ldo=ld)) == -1
    for rows in (0, 1):
        assert f(*attn_args(rows_k=rows, ldk=ld, ldv=ld)) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("ld", [0, 999, 1001, 4096, 1 << 33])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
def test_linear_rows(ld, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = lambda n: torch.randn(n, 1008, device="cuda", generator=g).to(dtype)[:, :999]  # noqa: E731
    A, W = rows(1), rows(300)
    want, got = torch.empty(1, 300, device="cuda"), torch.empty(1, 300, device="cuda")
    assert linear(A, W, want) == 0
    assert linear(A.as_strided((1, 999), (ld, 1)), W, got) == 0
    assert torch.equal(got, want)
    want, got = torch.empty(300, 1, device="cuda"), torch.empty(300, 1, device="cuda")
    assert linear(W, A, want) == 0
    assert linear(W, A.as_strided((1, 999), (ld, 1)), got) == 0
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("ld", [0, 129, 1 << 33])
def test_attention_rows(ld):
    g = torch.Generator(device="cuda").manual_seed(2)
    x, k, v = (torch.randn(r, 128, device="cuda", generator=g).to(torch.bfloat16) for r in (1, 90, 90))
    cu = lambda n: torch.tensor([0, n], dtype=torch.int32, device="cuda")  # noqa: E731
    one = lambda t: t.as_strided((1, 128), (ld, 1))  # noqa: E731
    want, got = torch.empty_like(x), torch.empty_like(x)
    assert attention(x, k, v, want, None, cu(1), cu(90), 1, 90, 2, 2, 64) == 0
    assert attention(one(x), k, v, one(got), None, cu(1), cu(90), 1, 90, 2, 2, 64) == 0
    assert torch.equal(got, want)
    q, many = torch.randn(100, 128, device="cuda", generator=g).to(torch.bfloat16), torch.empty(100, 128, device="cuda")
    many = many.to(torch.bfloat16)
    for rows in (1, 100):
        assert attention(q[:rows], one(x), one(x), many[:rows], None, cu(rows), cu(1), rows, 1, 2, 2, 64) == 0
        assert torch.equal(many[:rows], x.expand(rows, 128))
