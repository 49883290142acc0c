"""Measured cases of the layer operators: the norm with residual addition and 8-bit output, the matrix
product with bias, activation and residual in its epilogue, and the attention with capped scores,
distance bias, document and prefix masks.

``run`` computes a case in elementary torch operations in 32 bits where ``own`` is false, and through
the library's C entries (``laya_b200_norm``, ``laya_b200_linear``, ``laya_b200_attention_varlen``)
where it is true. ``exact`` restates each operator in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
CODE = {"bf16": 0, "fp16": 1, "fp32": 2, "e4m3": 3}  # LAYA_BF16 .. LAYA_E4M3 of the C header
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
ACT = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
E4M3_MAX = 448.0
FLT_MIN = 2.0 ** -126


def _norm(name, rows, D, x, resid, out, center=False, bias=False, keep=True, pad=0):
    return {"name": name, "op": "norm", "rows": rows, "D": D, "x": x, "resid": resid, "out": out, "center": center,
            "bias": bias, "keep": keep, "pad": pad}


def _linear(name, M, N, K, ab, out, act="none", bias=True, resid=False, pad=0):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "ab": ab, "out": out, "act": act, "bias": bias,
            "resid": resid, "pad": pad}


def _attn(name, B, lq, lk, Hq, Hkv, D, type, left=-1, right=-1, cap=0.0, slopes=False, prefix=0, docs=0, fused=False,
          lens=1):
    """lq, lk: "low high" of the lengths; lk "" means self-attention. docs: mean document length (0: no mask)."""
    return {"name": name, "op": "attn", "B": B, "lq": lq, "lk": lk, "Hq": Hq, "Hkv": Hkv, "D": D, "type": type,
            "left": left, "right": right, "cap": cap, "slopes": slopes, "prefix": prefix, "docs": docs,
            "fused": fused, "lens": lens}


def listed():
    return [
        # one new token between two layers: latency
        _norm("norm_token", 1, 1024, "bf16", "bf16", "e4m3"),
        # the packed benchmark batch (64 states x 3 questions): fp32 residual stream, LayerNorm, 8-bit output
        _norm("norm_batch", 52287, 1024, "bf16", "fp32", "e4m3", center=True),
        # a wide model's rows of odd width in padded storage, 16-bit output
        _norm("norm_wide_odd", 6007, 8191, "fp16", "fp16", "fp16", bias=True, pad=17),
        # MLP-in of one token: the weight is read once
        _linear("linear_token", 1, 5248, 1024, "bf16", "bf16", act="gelu"),
        # odd everything: a few questions' option rows through a classifier
        _linear("linear_odd", 77, 1153, 999, "fp16", "fp16", act="relu", resid=True, pad=1),
        # MLP-out of one 512-token question, 8-bit operands, added to the fp32 residual stream
        _linear("linear_question", 512, 1024, 2624, "e4m3", "fp32", resid=True),
        # MLP-out of the packed benchmark batch, 8-bit operands
        _linear("linear_batch", 52287, 1024, 2624, "e4m3", "bf16", resid=True, bias=False),
        # a wide layer over a long batch in 16 bits
        _linear("linear_wide", 16384, 8192, 4096, "fp16", "fp16", act="silu", resid=True),
        # one query row over one question's keys, scores biased by distance: latency
        _attn("attn_token", 1, "1 1", "512 512", 16, 16, 64, "bf16", slopes=True),
        # single-token serving over long ragged keys, shared key heads, capped scores
        _attn("attn_tokens_long", 24, "1 1", "1000 32768", 32, 8, 128, "bf16", cap=30.0),
        # the packed benchmark batch: every question holds several documents that do not see one another
        _attn("attn_batch_docs", 192, "32 512", "", 16, 16, 64, "bf16", docs=200, fused=True),
        # a long prompt whose prefix all tokens see, causal after it, capped scores
        _attn("attn_long_prefix", 1, "8192 8192", "", 16, 4, 128, "fp16", right=0, cap=50.0, prefix=1000),
    ]


def _spread(rng, low, high):
    """A whole number, uniform in its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "attn"])
    if op == "norm":
        D = _spread(rng, 64, 16384)
        if rng.random() < 0.5:
            D = max(64, D // 64 * 64)
        rows = _spread(rng, 1, max(1, min(60000, 36000000 // D)))
        c = _norm("", rows, D, rng.choice(["bf16", "fp16", "fp32"]), rng.choice(["", "bf16", "fp16", "fp32"]),
                  rng.choice(["bf16", "fp16", "fp32", "e4m3", "e4m3"]), center=rng.random() < 0.3,
                  bias=rng.random() < 0.3, keep=rng.random() < 0.7, pad=rng.choice([0, 0, 1, 8, 24]))
    elif op == "linear":
        M, N, K = _spread(rng, 1, 32768), _spread(rng, 16, 16384), _spread(rng, 16, 16384)
        if rng.random() < 0.6:
            N, K = max(16, N // 16 * 16), max(16, K // 16 * 16)
        while M * N * K > 16384 * 8192 * 4096 or M * N > 2 ** 28:
            M = (M + 1) // 2
        c = _linear("", M, N, K, rng.choice(["bf16", "fp16", "e4m3", "e4m3"]), rng.choice(["bf16", "fp16", "fp32"]),
                    act=rng.choice(list(ACT)), bias=rng.random() < 0.6, resid=rng.random() < 0.6,
                    pad=rng.choice([0, 0, 0, 3]))
    else:
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.choice([1, 2, 3, 4, 8])
        D = rng.choice([64, 128])
        if rng.random() < 0.4:  # few new rows over long keys
            high_q, high_k = rng.choice([1, 1, 2, 5]), _spread(rng, 64, 32768)
            B = _spread(rng, 1, 32)
            lk = "%d %d" % (rng.choice([1, max(1, high_k // 8), high_k]), high_k)
            lq = "%d %d" % (1, high_q)
        else:
            high_q = _spread(rng, 16, 8192)
            B = _spread(rng, 1, 128)
            lq, lk = "%d %d" % (rng.choice([0, 1, high_q // 2, high_q]), high_q), ""
            if rng.random() < 0.3:
                high_k = _spread(rng, high_q, 16384)
                lk = "%d %d" % (high_q, high_k)
            else:
                high_k = high_q
        while B * Hq * high_q * high_k > 16 * 8192 * 8192 // 2 or B * Hkv * high_k * D > 24 * 8 * 32768 * 128:
            if B > 1:
                B = (B + 1) // 2
            else:
                high_q = max(1, high_q // 2)
                lq = "%d %d" % (max(1, high_q // 2), high_q)
                if not lk:
                    high_k = high_q
        right = rng.choice([-1, -1, 0, 0, 64])
        left = rng.choice([-1, -1, -1, 64, 500])
        c = _attn("", B, lq, lk, Hq, Hkv, D, rng.choice(["bf16", "fp16"]), left=left, right=right,
                  cap=rng.choice([0.0, 0.0, 20.0, 50.0]), slopes=rng.random() < 0.3,
                  prefix=rng.choice([0, 0, 0, _spread(rng, 1, 2000)]), docs=rng.choice([0, 0, 0, 50, 1000]),
                  fused=not lk and rng.random() < 0.5, lens=rng.randrange(1 << 20))
    del c["name"]
    return c


# ------------------------------------------------------------------ what a case consists of
def _lengths(c):
    """Query and key lengths of every sequence, and the tokens' documents (-1: padding); from the case alone."""
    r = np.random.default_rng(c["lens"])
    low, high = map(int, c["lq"].split())
    lq = r.integers(low, high + 1, c["B"])
    lq[0] = high
    if c["lk"]:
        low, high = map(int, c["lk"].split())
        lk = np.maximum(r.integers(low, high + 1, c["B"]), 1)
        lk[0] = high
    else:
        lk = lq
    run = None
    if c["docs"]:  # for every key position: the start and end of its document, and whether it is padding
        run = []
        for n in lk:
            cuts = [0]
            while cuts[-1] < n:
                cuts.append(min(int(n), cuts[-1] + 1 + int(r.integers(0, 2 * c["docs"]))))
            pad = r.random(max(1, len(cuts) - 1)) < 0.03
            run.append((cuts, pad))
    return lq, lk, run


def _doc_ids(lq, lk, run):
    """Document ids of the key and the query tokens: query i of a sequence sits at key position i + lk - lq."""
    ks, qs = [], []
    for b, (cuts, pad) in enumerate(run):
        ids = np.zeros(int(lk[b]), np.int32)
        for d in range(len(cuts) - 1):
            ids[cuts[d]:cuts[d + 1]] = -1 if pad[d] else d
        at = np.arange(int(lq[b])) + int(lk[b]) - int(lq[b])
        ks.append(ids)
        qs.append(np.where(at >= 0, ids[np.maximum(at, 0)] if len(ids) else -1, -1).astype(np.int32))
    return np.concatenate(qs), np.concatenate(ks)


def _prefixes(c, lk):
    r = np.random.default_rng(c["lens"] + 1)
    return np.minimum(r.integers(c["prefix"] // 2, c["prefix"] + 1, len(lk)), lk).astype(np.int32)


def _pairs(c):
    """Query-key pairs that the masks leave, over all sequences."""
    lq, lk, run = _lengths(c)
    pre = _prefixes(c, lk) if c["prefix"] else np.zeros(len(lk), np.int64)
    n = 0
    for b in range(len(lq)):
        p = np.arange(int(lq[b])) + int(lk[b]) - int(lq[b])
        s, e = np.zeros_like(p), np.full_like(p, int(lk[b]))
        if run is not None:
            cuts, pad = run[b]
            if len(cuts) < 2:
                continue
            d = np.clip(np.searchsorted(cuts, p, side="right") - 1, 0, len(cuts) - 2)
            s, e = np.asarray(cuts)[d], np.asarray(cuts)[d + 1]
            e = np.where((p < 0) | pad[d], s, e)
        lo = np.maximum(s, p - c["left"]) if c["left"] >= 0 else s
        hi = np.minimum(e, p + c["right"] + 1) if c["right"] >= 0 else e
        in_window = np.maximum(0, hi - lo)
        x = np.minimum(e, int(pre[b]))
        in_prefix = np.maximum(0, x - s)
        both = np.maximum(0, np.minimum(hi, x) - lo)
        n += int((in_window + in_prefix - both).sum())
    return n


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["rows"] * c["D"]
        b = n * (SIZE[c["x"]] + (SIZE[c["resid"]] if c["resid"] else 0) + SIZE[c["out"]])
        b += n * _sum_size(c) + c["D"] * 4 * (2 if c["bias"] else 1) + (4 * c["rows"] if c["out"] == "e4m3" else 0)
        return {"bytes": b, "flops": 8 * n}
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        b = (M + N) * K * SIZE[c["ab"]] + M * N * SIZE[c["out"]] * (2 if c["resid"] else 1)
        b += 4 * N * c["bias"] + (4 * (M + N) if c["ab"] == "e4m3" else 0)
        return {"bytes": b, "flops": 2 * M * N * K}
    lq, lk, _ = _lengths(c)
    Tq, Tk = int(lq.sum()), int(lk.sum())
    b = 2 * c["D"] * (2 * Tq * c["Hq"] + 2 * Tk * c["Hkv"]) + 4 * Tq * c["Hq"] + (4 * (Tq + Tk) if c["docs"] else 0)
    return {"bytes": b, "flops": 4 * c["D"] * c["Hq"] * _pairs(c)}


def _sum_type(c):
    """The stored sum keeps the residual stream's type."""
    return c["resid"] if c["keep"] and c["resid"] else ""


def _sum_size(c):
    return SIZE[_sum_type(c)] if _sum_type(c) else 0


def _rows(g, rows, cols, dtype, pad, scale=1.0):
    """Random rows in storage of cols + pad columns."""
    t = torch.randn(rows, cols + pad, device="cuda", generator=g)
    return (t.mul_(scale)).to(dtype)[:, :cols]


def _empty(rows, cols, dtype, pad=0):
    return torch.empty(rows, cols + pad, device="cuda", dtype=dtype)[:, :cols]


def _quant(t):
    """Rows as e4m3 with a scale each, as weights and activations come to an 8-bit product."""
    s = (t.abs().amax(1) / E4M3_MAX).clamp_min(FLT_MIN)
    return (t / s[:, None]).to(torch.float8_e4m3fn), s


def _aligned(n, es):
    """Columns of storage that make rows of n values a multiple of 16 bytes."""
    return -(-n * es // 16) * 16 // es


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    if c["op"] == "norm":
        R, D = c["rows"], c["D"]
        c["tx"] = _rows(g, R, D, DT[c["x"]], c["pad"])
        c["tr"] = _rows(g, R, D, DT[c["resid"]], 0, 3.0) if c["resid"] else None
        c["w"] = 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
        c["b"] = 0.1 * torch.randn(D, device="cuda", generator=g) if c["bias"] else None
        c["tsum"] = _empty(R, D, DT[_sum_type(c)]) if _sum_type(c) else None
        c["tout"] = _empty(R, D, DT[c["out"]], c["pad"])
        c["scale"] = torch.empty(R, device="cuda") if c["out"] == "e4m3" else None
        return c
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        es = SIZE[c["ab"]]
        kp = _aligned(K, es) - K  # rows of A and W start on 16 bytes
        A = torch.randn(M, K + kp, device="cuda", generator=g)
        W = torch.randn(N, K + kp, device="cuda", generator=g) / math.sqrt(K)
        c["sa"] = c["sw"] = None
        if c["ab"] == "e4m3":
            (A, c["sa"]), (W, c["sw"]) = _quant(A), _quant(W)
        else:
            A, W = A.to(DT[c["ab"]]), W.to(DT[c["ab"]])
        c["A"], c["W"] = A[:, :K], W[:, :K]
        c["tbias"] = 0.5 * torch.randn(N, device="cuda", generator=g) if c["bias"] else None
        c["tres"] = _rows(g, M, N, DT[c["out"]], c["pad"]) if c["resid"] else None
        c["tout"] = _empty(M, N, DT[c["out"]], c["pad"])
        return c
    lq, lk, run = _lengths(c)
    Tq, Tk, Hq, Hkv, D = int(lq.sum()), int(lk.sum()), c["Hq"], c["Hkv"], c["D"]
    if c["fused"]:  # q | k | v of one projection's rows
        x = torch.randn(Tq, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(DT[c["type"]])
        c["q"], c["k"], c["v"] = x[:, :Hq * D], x[:, Hq * D:(Hq + Hkv) * D], x[:, (Hq + Hkv) * D:]
    else:
        c["q"] = torch.randn(Tq, Hq * D, device="cuda", generator=g).to(DT[c["type"]])
        c["k"] = torch.randn(Tk, Hkv * D, device="cuda", generator=g).to(DT[c["type"]])
        c["v"] = torch.randn(Tk, Hkv * D, device="cuda", generator=g).to(DT[c["type"]])
    cu = lambda n: torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).cuda()  # noqa: E731
    c["cuq"], c["cuk"] = cu(lq), cu(lk)
    c["mq"], c["mk"] = int(lq.max()), int(lk.max())
    c["tslopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device="cuda") if c["slopes"] else None
    c["tprefix"] = torch.from_numpy(_prefixes(c, lk)).cuda() if c["prefix"] else None
    c["dq"] = c["dk"] = None
    if run is not None:
        c["dq"], c["dk"] = (torch.from_numpy(t).cuda() for t in _doc_ids(lq, lk, run))
    c["tout"] = torch.empty(Tq, Hq * D, device="cuda", dtype=DT[c["type"]])
    c["lse"] = torch.empty(Tq, Hq, device="cuda")
    c["ws"] = None
    n = _workspace(c["B"], Tq, c["mq"], c["mk"], Hq, Hkv, D)
    if n:
        c["ws"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    return c


def _workspace(B, rows_q, max_q, max_k, Hq, Hkv, D):
    """Bytes of scratch that a program keeps for the joins of split keys: 32 partial rows for each row of
    a call with few rows, as laya_b200_attention_varlen_ws never asks for more."""
    return min(32 * rows_q * Hq * (D + 2) * 4, 1 << 28)


# ------------------------------------------------------------------ plain forms
def _plain_norm(c):
    h = c["tx"].float()
    if c["tr"] is not None:
        h = h + c["tr"].float()
    z = h - h.mean(1, keepdim=True) if c["center"] else h
    y = z * torch.rsqrt((z * z).mean(1, keepdim=True) + 1e-5) * c["w"]
    if c["b"] is not None:
        y = y + c["b"]
    r = {}
    if c["tsum"] is not None:
        r["sum"] = h.to(c["tsum"].dtype)
    if c["scale"] is not None:
        s = (y.abs().amax(1) / E4M3_MAX).clamp_min(FLT_MIN)
        r["scale"], y = s, y / s[:, None]
    r["out"] = y.to(c["tout"].dtype)
    return r


def _act(y, act):
    if act == "relu":
        return torch.clamp_min(y, 0)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    return y


def _plain_linear(c):
    y = c["A"].float() @ c["W"].float().t()
    if c["sa"] is not None:
        y = y * c["sa"][:, None] * c["sw"]
    if c["tbias"] is not None:
        y = y + c["tbias"]
    y = _act(y, c["act"])
    if c["tres"] is not None:
        y = y + c["tres"].float()
    return {"out": y.to(c["tout"].dtype)}


def _plain_attn(c):
    """Every sequence padded to the longest; the scores of all pairs at once."""
    B, Hq, Hkv, D, mq, mk = c["B"], c["Hq"], c["Hkv"], c["D"], c["mq"], c["mk"]
    dev = c["q"].device
    cuq, cuk = c["cuq"].long(), c["cuk"].long()
    lq, lk = cuq[1:] - cuq[:-1], cuk[1:] - cuk[:-1]
    i, j = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
    rows_q, rows_k = max(1, c["q"].shape[0]), max(1, c["k"].shape[0])
    at_q = (cuq[:-1, None] + i).clamp_max(rows_q - 1)
    at_k = (cuk[:-1, None] + j).clamp_max(rows_k - 1)
    G = Hq // Hkv
    q = c["q"].float()[at_q].view(B, mq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * mq, D)
    k = c["k"].float()[at_k].view(B, mk, Hkv, D).permute(0, 2, 3, 1)
    v = c["v"].float()[at_k].view(B, mk, Hkv, D).permute(0, 2, 1, 3)
    s = (q @ k).view(B, Hkv, G, mq, mk) * (D ** -0.5)
    if c["cap"]:
        s = c["cap"] * torch.tanh(s / c["cap"])
    p = i + (lk - lq)[:, None]  # [B, mq]: the query rows' positions among the keys
    away = p[:, :, None] - j  # [B, mq, mk]
    if c["tslopes"] is not None:
        s = s - c["tslopes"].view(1, Hkv, G, 1, 1) * away.abs().float()[:, None, None]
    see = torch.ones_like(away, dtype=torch.bool)
    if c["left"] >= 0:
        see &= away <= c["left"]
    if c["right"] >= 0:
        see &= -away <= c["right"]
    if c["tprefix"] is not None:
        see |= j < c["tprefix"].long()[:, None, None]
    see &= j < lk[:, None, None]
    if c["dq"] is not None:
        dq, dk = c["dq"][at_q], c["dk"][at_k]
        see &= (dq[:, :, None] == dk[:, None, :]) & (dk >= 0)[:, None, :]
    s = s.masked_fill(~see[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True).clamp_min(-3e38)
    s = torch.exp(s - m)
    l = s.sum(-1, keepdim=True)
    o = (s.view(B, Hkv, G * mq, mk) @ v).view(B, Hkv, G, mq, D) / l.clamp_min(1e-30)
    lse = (m + torch.log(l)).squeeze(-1)
    t = torch.arange(c["q"].shape[0], device=dev)
    b = torch.searchsorted(cuq, t, right=True) - 1
    o = o.permute(0, 3, 1, 2, 4).reshape(B, mq, Hq * D)[b, t - cuq[b]]
    lse = lse.permute(0, 3, 1, 2).reshape(B, mq, Hq)[b, t - cuq[b]]
    return {"out": o.to(c["tout"].dtype), "lse": lse}


# ------------------------------------------------------------------ the library's entries
def _ptr(t):
    return None if t is None else t.data_ptr()


def _ld(t):
    return 0 if t is None else t.stride(0)


def _ok(rc, what):
    if rc != 0:
        raise RuntimeError("%s returned %d" % (what, rc))


def _own_norm(L, st, c):
    _ok(L.laya_b200_norm(_ptr(c["tx"]), CODE[c["x"]], _ld(c["tx"]), _ptr(c["tr"]), CODE[c["resid"] or c["x"]],
                         _ld(c["tr"]), _ptr(c["tsum"]), CODE[_sum_type(c) or c["x"]], _ld(c["tsum"]), _ptr(c["w"]),
                         _ptr(c["b"]), 1e-5, int(c["center"]), _ptr(c["tout"]), CODE[c["out"]], _ld(c["tout"]),
                         _ptr(c["scale"]), c["rows"], c["D"], st, 0), "laya_b200_norm")
    r = {"out": c["tout"]}
    if c["tsum"] is not None:
        r["sum"] = c["tsum"]
    if c["scale"] is not None:
        r["scale"] = c["scale"]
    return r


def _own_linear(L, st, c):
    _ok(L.laya_b200_linear(_ptr(c["A"]), _ld(c["A"]), _ptr(c["W"]), _ld(c["W"]), CODE[c["ab"]], _ptr(c["sa"]),
                           _ptr(c["sw"]), _ptr(c["tbias"]), ACT[c["act"]], _ptr(c["tres"]), _ld(c["tres"]),
                           _ptr(c["tout"]), CODE[c["out"]], _ld(c["tout"]), c["M"], c["N"], c["K"], st, 0),
        "laya_b200_linear")
    return {"out": c["tout"]}


def _own_attn(L, st, c):
    _ok(L.laya_b200_attention_varlen(
        _ptr(c["q"]), _ld(c["q"]), _ptr(c["k"]), _ld(c["k"]), _ptr(c["v"]), _ld(c["v"]), _ptr(c["tout"]),
        _ld(c["tout"]), _ptr(c["lse"]), CODE[c["type"]], _ptr(c["cuq"]), _ptr(c["cuk"]), c["B"], c["q"].shape[0],
        c["k"].shape[0], c["mq"], c["mk"], c["Hq"], c["Hkv"], c["D"], c["D"] ** -0.5, c["cap"], _ptr(c["tslopes"]),
        c["left"], c["right"], _ptr(c["tprefix"]), _ptr(c["dq"]), _ptr(c["dk"]), _ptr(c["ws"]),
        0 if c["ws"] is None else c["ws"].numel(), st, 0), "laya_b200_attention_varlen")
    return {"out": c["tout"], "lse": c["lse"]}


def run(state):
    c = state
    if own:
        from layamd_b200 import load_lib
        call = {"norm": _own_norm, "linear": _own_linear, "attn": _own_attn}[c["op"]]
        return call(load_lib(), torch.cuda.current_stream().cuda_stream, c)
    return {"norm": _plain_norm, "linear": _plain_linear, "attn": _plain_attn}[c["op"]](c)


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    c = prepare(case, seed)
    f = torch.float64
    if c["op"] == "norm":
        h = c["tx"].to(f) + (c["tr"].to(f) if c["tr"] is not None else 0)
        mean = h.sum(1) / c["D"] if c["center"] else torch.zeros(c["rows"], dtype=f, device="cuda")
        var = (h - mean[:, None]).pow(2).sum(1) / c["D"]
        y = (h - mean[:, None]) / torch.sqrt(var + 1e-5)[:, None] * c["w"].to(f)
        y = y + c["b"].to(f) if c["b"] is not None else y
        r = {"out": y}
        if c["scale"] is not None:
            r["scale"] = torch.maximum(y.abs().max(1).values / E4M3_MAX, torch.full_like(mean, FLT_MIN))
            r["out"] = y / r["scale"][:, None]  # before its rounding to 8 bits
        if c["tsum"] is not None:
            r["sum"] = h
        return r
    if c["op"] == "linear":
        y = torch.matmul(c["A"].to(f), c["W"].to(f).T)
        if c["sa"] is not None:
            y = c["sa"].to(f)[:, None] * y * c["sw"].to(f)[None]
        if c["tbias"] is not None:
            y += c["tbias"].to(f)
        if c["act"] == "relu":
            y = torch.where(y > 0, y, torch.zeros_like(y))
        elif c["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        elif c["act"] == "silu":
            y = y * torch.sigmoid(y)
        return {"out": y + c["tres"].to(f) if c["tres"] is not None else y}
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    cuq, cuk = c["cuq"].tolist(), c["cuk"].tolist()
    out = torch.zeros(cuq[-1], Hq, D, dtype=f, device="cuda")
    lse = torch.full((cuq[-1], Hq), -math.inf, dtype=f, device="cuda")
    for b in range(c["B"]):
        n, m = cuq[b + 1] - cuq[b], cuk[b + 1] - cuk[b]
        if not n or not m:
            continue
        q = c["q"][cuq[b]:cuq[b + 1]].to(f).view(n, Hkv, Hq // Hkv, D)
        k = c["k"][cuk[b]:cuk[b + 1]].to(f).view(m, Hkv, D)
        v = c["v"][cuk[b]:cuk[b + 1]].to(f).view(m, Hkv, D)
        s = torch.einsum("nhgd,mhd->hgnm", q, k) / math.sqrt(D)
        if c["cap"]:
            s = torch.tanh(s / c["cap"]) * c["cap"]
        pos, key = torch.arange(m - n, m, device="cuda")[:, None], torch.arange(m, device="cuda")[None]
        if c["slopes"]:
            slope = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device="cuda").to(f)
            s -= slope.view(Hkv, Hq // Hkv, 1, 1) * (pos - key).abs()
        hidden = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        if c["left"] >= 0:
            hidden |= key < pos - c["left"]
        if c["right"] >= 0:
            hidden |= key > pos + c["right"]
        if c["prefix"]:
            hidden &= key >= c["tprefix"][b]
        if c["docs"]:
            a, d = c["dq"][cuq[b]:cuq[b + 1], None], c["dk"][None, cuk[b]:cuk[b + 1]]
            hidden |= (a != d) | (d < 0)
        s.masked_fill_(hidden, -math.inf)
        z = torch.logsumexp(s, -1)
        w = torch.exp_(s.sub_(torch.where(z.isinf(), torch.zeros_like(z), z)[..., None]))
        out[cuq[b]:cuq[b + 1]] = torch.einsum("hgnm,mhd->nhgd", w, v).reshape(n, Hq, D)
        lse[cuq[b]:cuq[b + 1]] = z.permute(2, 0, 1).reshape(n, Hq)
    return {"out": out.view(-1, Hq * D), "lse": lse}


if __name__ == "__main__":  # the cases and their work
    rng = random.Random(0)
    for case in listed() + [draw(rng) for _ in range(4)]:
        print(case.get("name", "drawn"), work(case))
