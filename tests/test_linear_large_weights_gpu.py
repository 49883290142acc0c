"""laya_b200_linear with few rows and large weights, where its kernels take over from one another: against the
formula in 64 bits, with the bounds of the product's tests."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_linear_gpu import BF, E4, HF, F32, case, gpu  # noqa: E402, F401


@pytest.mark.parametrize("M", [1, 3, 4, 7, 8, 15, 16, 17])
@pytest.mark.parametrize("ab,N,K", [
    (BF, 1801, 28672), (E4, 1760, 57344), (BF, 1760, 28656),  # rows of 56 KB, and a little shorter
    (BF, 3100, 16384), (HF, 6150, 8192), (E4, 12300, 8192),   # 32, 16 and 8 KB
    (BF, 9472, 5400), (HF, 16385, 4000)])                     # many columns
def test_large_weights(M, N, K, ab):
    case(M, N, K, ab, BF if M < 8 else F32, scales=ab == E4, bias=True, act=3, resid=True)
