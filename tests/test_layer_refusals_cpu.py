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


def attn_args(**kw):
    a = dict(q=A, ldq=256, k=A, ldk=128, v=A, ldv=128, out=A, ldo=256, lse=A, type=BF16, cu_q=A, cu_k=A, B=2, rows_q=8,
             rows_k=9, max_q=4, max_k=5, Hq=4, Hkv=2, D=64, scale=0.125, softcap=0.0, slopes=A, left=-1, right=0,
             prefix=A, doc_q=A, doc_k=A, ws=None, ws_bytes=0, stream=None, sync=0)
    a.update(kw)
    return list(a.values())


def test_attention_accepts(L):
    f = L.laya_b200_attention_varlen
    assert f(*attn_args()) == -1
    assert f(*attn_args(lse=None, slopes=None, prefix=None, doc_q=None, doc_k=None)) == -1
    assert f(*attn_args(rows_q=1, ldq=0, ldo=0, rows_k=1, ldk=0, ldv=0)) == -1
    assert f(*attn_args(rows_k=0, k=None, v=None, ldk=0, ldv=0)) == -1
    assert f(*attn_args(B=0)) == 0 and f(*attn_args(rows_q=0)) == 0 and f(*attn_args(max_q=0)) == 0
    assert L.laya_b200_attention_varlen_ws(2, 8, 4, 5, 4, 2, 64) == -1


@pytest.mark.parametrize("kw", [
    dict(type=F32), dict(type=E4M3), dict(D=32), dict(D=96), dict(Hq=3), dict(Hkv=0), dict(Hq=2, Hkv=4),
    dict(Hq=2048, Hkv=2), dict(B=-1), dict(B=65536), dict(rows_q=-1), dict(rows_k=-1), dict(rows_q=(1 << 29) + 1),
    dict(max_q=-1), dict(max_k=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("nan")), dict(softcap=1e-41),
    dict(scale=1e-30, softcap=1e15), dict(left=-2), dict(right=-2),
    dict(doc_q=None), dict(doc_k=None), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu_q=None),
    dict(cu_k=None), dict(ldq=248), dict(ldq=260), dict(ldk=120), dict(ldv=129), dict(ldo=255), dict(ldo=1 << 33),
    dict(q=A + 8), dict(k=A + 2), dict(v=A + 8), dict(out=A + 4), dict(lse=A + 2), dict(cu_q=A + 1), dict(ws=A + 8),
    dict(ws_bytes=-1)])
def test_attention_refuses(L, kw):
    assert L.laya_b200_attention_varlen(*attn_args(**kw)) == -2


def test_attention_workspace_refuses(L):
    f = L.laya_b200_attention_varlen_ws
    assert f(-1, 8, 4, 5, 4, 2, 64) == -2 and f(2, 8, 4, 5, 4, 3, 64) == -2 and f(2, 8, 4, 5, 4, 2, 80) == -2
