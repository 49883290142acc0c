"""Calls of the layer operators' C entries on torch tensors, for their tests."""
import torch

from layamd_b200 import load_lib

CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, torch.float8_e4m3fn: 3}


def ptr(t):
    return None if t is None else t.data_ptr()


def code(t, default=0):
    return default if t is None else CODE[t.dtype]


def ld(t):
    return 0 if t is None else t.stride(0)


def half_step(dtype):
    """Largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


def stream():
    return torch.cuda.current_stream().cuda_stream if torch.cuda.is_available() else None


def norm(x, w, out, resid=None, sum=None, b=None, scale=None, eps=1e-5, center=0, sync=1, rows=None, D=None):
    return load_lib().laya_b200_norm(ptr(x), code(x), ld(x), ptr(resid), code(resid), ld(resid), ptr(sum), code(sum),
                                     ld(sum), ptr(w), ptr(b), eps, center, ptr(out), code(out), ld(out), ptr(scale),
                                     x.shape[0] if rows is None else rows, x.shape[1] if D is None else D, stream(),
                                     sync)


def linear(A, W, out, a_scale=None, w_scale=None, bias=None, act=0, resid=None, sync=1, M=None, N=None, K=None):
    return load_lib().laya_b200_linear(ptr(A), ld(A), ptr(W), ld(W), code(A), ptr(a_scale), ptr(w_scale), ptr(bias),
                                       act, ptr(resid), ld(resid), ptr(out), code(out), ld(out),
                                       A.shape[0] if M is None else M, W.shape[0] if N is None else N,
                                       A.shape[1] if K is None else K, stream(), sync)


def attention(q, k, v, out, lse, cu_q, cu_k, max_q, max_k, Hq, Hkv, D, scale=None, cap=0.0, slopes=None, left=-1,
              right=-1, prefix=None, doc_q=None, doc_k=None, ws=None, sync=1):
    return load_lib().laya_b200_attention_varlen(
        ptr(q), ld(q), ptr(k), ld(k), ptr(v), ld(v), ptr(out), ld(out), ptr(lse), code(q), ptr(cu_q), ptr(cu_k),
        cu_q.numel() - 1, q.shape[0], k.shape[0], max_q, max_k, Hq, Hkv, D, D ** -0.5 if scale is None else scale, cap,
        ptr(slopes), left, right, ptr(prefix), ptr(doc_q), ptr(doc_k), ptr(ws), 0 if ws is None else ws.numel(),
        stream(), sync)
