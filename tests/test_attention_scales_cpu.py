"""Scales and caps that laya_b200_attention_varlen takes, without a GPU: accepted ones get as far as the missing
device (-1)."""
import pytest

from tests.test_layer_refusals_cpu import L, attn_args  # noqa: F401


@pytest.mark.parametrize("scale,cap,rc", [
    (2.0 ** 126, 0.0, -1), (2.0 ** 126, 2.0 ** 126, -1), (1e-37, 0.0, -1), (1.0, 2.0 ** 126, -1), (1.0, 1e-30, -1),
    (1e38, 0.0, -2), (3e38, 3e38, -2), (1.0, 1e38, -2), (1.0, 3e38, -2)])
def test_scales(L, scale, cap, rc):  # noqa: F811
    """Above 2^126 the product with log2 e, in which the softmax is computed, leaves fp32's range."""
    assert L.laya_b200_attention_varlen(*attn_args(scale=scale, softcap=cap)) == rc
