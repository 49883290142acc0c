"""laya_b200_attention_varlen on either side of the border between its kernels (8 queries), with any number of
query heads to a key head: against the formula in 64 bits, with the bounds of the attention tests."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from tests.test_attention_varlen_gpu import HF, gpu, run  # noqa: E402, F401


@pytest.mark.parametrize("lq", [1, 7, 8, 9])
@pytest.mark.parametrize("G", [1, 3, 16, 130])
@pytest.mark.parametrize("D", [64, 128])
def test_border(lq, G, D):
    run([lq, 1, 0], [300, 77, 5], D=D, Hq=G, Hkv=1, right=0)
    run([lq], [700], D=D, Hq=2 * G, Hkv=2, left=90, prefix=[40], dtype=HF, cap=20.0)
    ids = [i // 30 if i % 11 else -2 for i in range(200)]
    run([lq], [200], D=D, Hq=G, Hkv=1, docs=([ids[-lq:]], [ids]))
    run([lq], [2500], D=D, Hq=G, Hkv=1, slopes=True)
    run([lq], [2500], D=D, Hq=G, Hkv=1, ws="none")
