"""How many sequences, rows and heads a laya_b200_attention_varlen call may have, without a GPU: accepted
arguments get as far as the missing device (-1)."""
from tests.test_layer_refusals_cpu import L, attn_args  # noqa: F401


def test_sizes(L):  # noqa: F811
    f, ws = L.laya_b200_attention_varlen, L.laya_b200_attention_varlen_ws
    big = 1 << 29
    for kw in (dict(B=65535, rows_q=131070, max_q=65536, Hq=64, Hkv=1),  # one long sequence among single tokens
               dict(B=65535, rows_q=1 << 24, max_q=1 << 24, Hq=128, Hkv=1),
               dict(B=1, rows_q=big, max_q=big, Hq=64, Hkv=1), dict(B=512, rows_q=65536, max_q=big)):
        a = attn_args(**kw)
        if "Hkv" in kw:
            a = attn_args(**kw, ldq=64 * kw["Hq"], ldo=64 * kw["Hq"], ldk=64, ldv=64)
        assert f(*a) == -1
    # 2^31 units of work and more: rows and heads that no GPU holds
    a = dict(B=65535, rows_q=big, max_q=big, Hq=1024, Hkv=1, ldq=65536, ldo=65536)
    assert f(*attn_args(**a)) == -2
    assert ws(65535, big, big, 5, 1024, 1, 64) == -2 and ws(65535, big, 5, 5, 1024, 1, 64) == -1
