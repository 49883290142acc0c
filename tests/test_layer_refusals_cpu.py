"""Arguments that the layer operators refuse, without a GPU: the checks come before any CUDA call, so a
refused argument gives -2 and an accepted one gets as far as the missing device (-1)."""
import pytest

torch = pytest.importorskip("torch")

from layamd_b200 import load_lib

BF16, F16, F32, E4M3 = 0, 1, 2, 3
A = 1 << 20  # an address that nothing reads: every call here ends before a launch


@pytest.fixture(scope="module")
def L():
    if torch.cuda.is_available():
        pytest.skip("made-up addresses: only where there is no GPU")
    return load_lib()


def norm_args(**kw):
    a = dict(x=A, x_type=BF16, ldx=64, resid=A, resid_type=F32, ldr=64, sum=A, sum_type=F32, lds=64, w=A, b=A,
             eps=1e-5, center=0, out=A, out_type=E4M3, ldo=64, scale=A, rows=4, D=64, stream=None, sync=0)
    a.update(kw)
    return list(a.values())


def test_norm_accepts(L):
    assert L.laya_b200_norm(*norm_args()) == -1
    assert L.laya_b200_norm(*norm_args(resid=None, resid_type=9, sum=None, sum_type=9, b=None)) == -1
    assert L.laya_b200_norm(*norm_args(rows=1, ldx=0, ldr=0, lds=0, ldo=0)) == -1
    assert L.laya_b200_norm(*norm_args(out_type=F32, scale=None)) == -1
    assert L.laya_b200_norm(*norm_args(rows=0, x=None, out=None)) == 0


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(D=0), dict(D=16385, ldx=20000, ldr=20000, lds=20000, ldo=20000), dict(x_type=E4M3),
    dict(x_type=-1), dict(resid_type=E4M3), dict(sum_type=E4M3), dict(sum_type=4), dict(out_type=4), dict(center=2),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(x=None), dict(w=None), dict(out=None),
    dict(scale=None), dict(out_type=BF16), dict(ldx=63), dict(ldr=63), dict(lds=63), dict(ldo=63), dict(ldx=-64),
    dict(x=A + 1), dict(resid=A + 2), dict(sum=A + 2), dict(w=A + 2), dict(b=A + 1), dict(scale=A + 2)])
def test_norm_refuses(L, kw):
    assert L.laya_b200_norm(*norm_args(**kw)) == -2


def linear_args(**kw):
    a = dict(A=A, lda=64, W=A, ldw=64, ab_type=BF16, a_scale=A, w_scale=A, bias=A, act=2, resid=A, ldr=24, out=A,
             out_type=F32, ldo=24, M=8, N=24, K=64, stream=None, sync=0)
    a.update(kw)
    return list(a.values())


def test_linear_accepts(L):
    assert L.laya_b200_linear(*linear_args()) == -1
    assert L.laya_b200_linear(*linear_args(a_scale=None, w_scale=None, bias=None, resid=None, ldr=0)) == -1
    assert L.laya_b200_linear(*linear_args(K=63, N=23)) == -1
    assert L.laya_b200_linear(*linear_args(M=1, lda=0, ldo=0, ldr=0)) == -1
    assert L.laya_b200_linear(*linear_args(ab_type=E4M3, K=50)) == -1
    assert L.laya_b200_linear(*linear_args(out=A + 4, resid=A + 4, ldo=25, ldr=27)) == -1
    assert L.laya_b200_linear(*linear_args(M=0, A=None)) == 0
    assert L.laya_b200_linear(*linear_args(N=0, W=None)) == 0


@pytest.mark.parametrize("kw", [
    dict(M=-1), dict(N=-1), dict(K=0), dict(K=(1 << 24) + 1, lda=1 << 25, ldw=1 << 25), dict(ab_type=F32),
    dict(ab_type=4), dict(out_type=E4M3), dict(out_type=-1), dict(act=4), dict(act=-1), dict(A=None), dict(W=None),
    dict(out=None), dict(lda=63), dict(lda=66), dict(ldw=68), dict(ldw=56), dict(lda=-64), dict(lda=1 << 33),
    dict(A=A + 8), dict(W=A + 2), dict(ldo=23), dict(ldr=23), dict(out=A + 2), dict(resid=A + 2), dict(bias=A + 2),
    dict(a_scale=A + 1), dict(w_scale=A + 3), dict(ab_type=E4M3, lda=72, ldw=72)])
def test_linear_refuses(L, kw):
    assert L.laya_b200_linear(*linear_args(**kw)) == -2
