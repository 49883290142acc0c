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
