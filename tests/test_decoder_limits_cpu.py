"""Sizes that the decoder-layer kernels' 32-bit counts do not hold are refused before anything is launched."""
import ctypes

import pytest
import torch

from apnn_tc_b200 import _cabi
from test_decoder_cpu import P, UNSUPPORTED, batch, cache, linear

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("kw", [dict(M=TOP), dict(M=TOP - 255), dict(N=TOP, ldo=TOP, wbits=1), dict(N=TOP // 2, ldo=TOP, wbits=2),
                                dict(N=TOP - 255, ldo=TOP, wbits=1), dict(K=TOP, ldx=2 ** 31), dict(K=TOP - 511, ldx=2 ** 31), dict(M=1, K=TOP - 100, ldx=2 ** 31)])
def test_product_sizes(kw):
    assert linear(**kw) == UNSUPPORTED


def append(c, b, **kw):
    a = _cabi.Kv4AppendArgs(**{**dict(rows=2, k=P, v=P, k_stride=1 << 40, v_stride=1 << 40, eps=1e-6), **kw})
    return _cabi.lib().apnn_kv4_append(None, ctypes.addressof(c), ctypes.addressof(b), ctypes.addressof(a))


def attention(c, b, **kw):
    a = _cabi.Kv4AttentionArgs(**{**dict(rows=2, q=P, out=P, q_stride=1 << 40, out_stride=1 << 40, q_heads=4, causal=1, scale=0.1), **kw})
    return _cabi.lib().apnn_kv4_attention(None, ctypes.addressof(c), ctypes.addressof(b), ctypes.addressof(a), P, 1 << 60)


@pytest.mark.parametrize("heads", [(1 << 20) + 1, 1 << 28, TOP])
def test_heads(heads):
    L, b = _cabi.lib(), batch()
    wide = cache(heads=heads, page_stride=1 << 44)
    assert append(wide, b) == UNSUPPORTED
    assert L.apnn_kv4_read(None, ctypes.addressof(wide), ctypes.addressof(b), P, P, 2) == UNSUPPORTED
    assert attention(wide, b, q_heads=heads, q_stride=1 << 40, out_stride=1 << 40) == UNSUPPORTED
    c = cache(heads=1)
    assert append(c, b, q=P, q_out=P, q_heads=heads, q_stride=1 << 40, q_out_stride=1 << 40) == UNSUPPORTED
    assert attention(c, b, q_heads=heads, q_stride=1 << 40, out_stride=1 << 40) == UNSUPPORTED
    assert L.apnn_kv4_attention_workspace_bytes(ctypes.addressof(c), ctypes.addressof(b), heads) == 0


@pytest.mark.parametrize("head_dim,most", [(64, 65535 * 256), (128, 65535 * 256), (256, 65535 * 128)])
def test_rows_of_a_sequence(head_dim, most):
    c = cache(head_dim=head_dim, page_stride=1 << 16)
    for max_q in (most // 2 + 1, 1 << 30):      # two query heads to a key head
        assert attention(c, batch(max_q=max_q)) == UNSUPPORTED


def test_check_of_a_host_tensor():
    import apnn_tc_b200 as ap
    with pytest.raises(ValueError, match="CUDA"):
        ap.kv4_attention_check(torch.zeros(64, dtype=torch.uint8))
