"""The decoder-layer entry points refuse what they cannot do, before they touch a device; the plain forms agree with themselves."""
import ctypes

import numpy as np
import pytest
import torch

import decoder_reference as ref
from apnn_tc_b200 import _cabi

BUF = (ctypes.c_uint32 * 4096)()
P = ctypes.addressof(BUF) + (-ctypes.addressof(BUF) % 16)
INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE = 1, 2, 3, 4


def linear(wbits=4, W=P, X=P, Out=P, M=4, N=64, K=128, flag=None, **kw):
    d = dict(x_type=0, out_type=0, activation=0, zero=7.5, scale=P, ldx=K, ldo=N)
    d.update(kw)
    size = d.pop("struct_size", None)
    desc = _cabi.LinearDesc(**d)
    if size is not None:
        desc.struct_size = size
    return _cabi.lib().apnn_linear_planes(None, wbits, W, X, Out, M, N, K, ctypes.addressof(desc), flag)


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(W=None)), (INVALID, dict(X=None)), (INVALID, dict(Out=None)), (INVALID, dict(scale=None)),
    (INVALID, dict(M=0)), (INVALID, dict(N=-1)), (INVALID, dict(K=0)), (INVALID, dict(struct_size=8)),
    (INVALID, dict(x_type=2)), (INVALID, dict(out_type=1)), (INVALID, dict(activation=5)), (INVALID, dict(zero=0.25)),
    (INVALID, dict(zero=-0.5)), (INVALID, dict(zero=15.5)), (INVALID, dict(zero=float("nan"))), (INVALID, dict(ldx=120)),
    (INVALID, dict(ldo=63)), (INVALID, dict(residual=P, ldr=63)),
    (UNSUPPORTED, dict(wbits=0)), (UNSUPPORTED, dict(wbits=5)), (UNSUPPORTED, dict(wbits=8)),
    (UNSUPPORTED, dict(N=1 << 30, ldo=1 << 30)),
    (ALIGNMENT, dict(W=P + 4)), (ALIGNMENT, dict(X=P + 2)), (ALIGNMENT, dict(ldx=132)), (ALIGNMENT, dict(Out=P + 1)),
    (ALIGNMENT, dict(out_type=2, Out=P + 2)), (ALIGNMENT, dict(scale=P + 2)), (ALIGNMENT, dict(flag=P + 1)),
])
def test_linear_refuses(status, kw):
    assert linear(**kw) == status


def cache(**kw):
    d = dict(type=0, data=P, page_stride=16 * 72 * 2, pages=4, heads=2, page_size=16, head_dim=64)
    d.update(kw)
    return _cabi.Kv4Cache(**d)


def batch(**kw):
    d = dict(sequences=2, cu_q=P, kv_len=P, table=P, table_stride=3, table_width=3, max_q=1)
    d.update(kw)
    return _cabi.Kv4Batch(**d)


def each(c, b):
    """The three calls on this cache and batch, otherwise valid."""
    L = _cabi.lib()
    a = _cabi.Kv4AppendArgs(rows=2, k=P, v=P, k_stride=128, v_stride=128, eps=1e-6)
    t = _cabi.Kv4AttentionArgs(rows=2, q=P, out=P, q_stride=256, out_stride=256, q_heads=4, causal=1, scale=0.1)
    c, b = ctypes.addressof(c), ctypes.addressof(b)
    return (L.apnn_kv4_append(None, c, b, ctypes.addressof(a)), L.apnn_kv4_read(None, c, b, P, P, 2),
            L.apnn_kv4_attention(None, c, b, ctypes.addressof(t), P, 1 << 40))


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(data=None)), (INVALID, dict(type=2)), (INVALID, dict(pages=0)), (INVALID, dict(heads=0)),
    (INVALID, dict(page_stride=16 * 72)), (UNSUPPORTED, dict(head_dim=96)), (UNSUPPORTED, dict(head_dim=512)),
    (UNSUPPORTED, dict(page_size=24)), (UNSUPPORTED, dict(page_size=4)), (UNSUPPORTED, dict(page_size=2048)),
    (ALIGNMENT, dict(data=P + 8)), (ALIGNMENT, dict(page_stride=16 * 72 * 2 + 8)),
])
def test_cache_refused(status, kw):
    assert each(cache(**kw), batch()) == (status,) * 3


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(cu_q=None)), (INVALID, dict(kv_len=None)), (INVALID, dict(table=None)), (INVALID, dict(sequences=0)),
    (INVALID, dict(table_width=0)), (INVALID, dict(table_stride=2)), (INVALID, dict(max_q=0)), (ALIGNMENT, dict(cu_q=P + 2)),
])
def test_batch_refused(status, kw):
    assert each(cache(), batch(**kw)) == (status,) * 3


def test_descriptors_of_another_size_are_refused():
    for which in (0, 1):
        c, b = cache(), batch()
        (c, b)[which].struct_size = 8
        assert each(c, b) == (INVALID,) * 3


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(rows=0)), (INVALID, dict(k=None)), (INVALID, dict(v=None)), (INVALID, dict(k_stride=120)), (INVALID, dict(q=P)),
    (INVALID, dict(q=P, q_out=P, q_heads=0)), (INVALID, dict(q=P, q_out=P, q_heads=2, q_stride=64, q_out_stride=128)),
    (INVALID, dict(rotary_dim=32)), (INVALID, dict(rotary=P, rotary_rows=0, rotary_dim=32)), (INVALID, dict(rotary=P, rotary_rows=4, rotary_dim=80)),
    (UNSUPPORTED, dict(rotary=P, rotary_rows=4, rotary_dim=24)), (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=float("nan"))),
    (INVALID, dict(interleaved=2)), (ALIGNMENT, dict(k=P + 2)), (ALIGNMENT, dict(v_stride=132)), (ALIGNMENT, dict(k_norm=P + 8)),
    (ALIGNMENT, dict(rotary=P + 8, rotary_rows=4, rotary_dim=32)),
])
def test_append_refuses(status, kw):
    d = dict(rows=2, k=P, v=P, k_stride=128, v_stride=128, eps=1e-6)
    d.update(kw)
    c, b, a = cache(), batch(), _cabi.Kv4AppendArgs(**d)
    assert _cabi.lib().apnn_kv4_append(None, ctypes.addressof(c), ctypes.addressof(b), ctypes.addressof(a)) == status


@pytest.mark.parametrize("status,kw", [
    (INVALID, dict(rows=-1)), (INVALID, dict(q=None)), (INVALID, dict(out=None)), (INVALID, dict(q_heads=3)), (INVALID, dict(q_heads=0)),
    (INVALID, dict(q_stride=128)), (INVALID, dict(causal=2)), (INVALID, dict(window=-1)), (INVALID, dict(causal=0, window=8)),
    (INVALID, dict(scale=float("inf"))), (ALIGNMENT, dict(q=P + 4)), (ALIGNMENT, dict(out_stride=260)), (ALIGNMENT, dict(lse=P + 2)),
])
def test_attention_refuses(status, kw):
    d = dict(rows=2, q=P, out=P, q_stride=256, out_stride=256, q_heads=4, causal=1, scale=0.1)
    d.update(kw)
    c, b, a = cache(), batch(), _cabi.Kv4AttentionArgs(**d)
    assert _cabi.lib().apnn_kv4_attention(None, ctypes.addressof(c), ctypes.addressof(b), ctypes.addressof(a), P, 1 << 40) == status


@pytest.mark.parametrize("kw", [dict(table_width=(1 << 30) // 8 + 1), dict(sequences=1 << 12, table_width=1 << 24)])
def test_attention_refuses_what_32_bits_do_not_count(kw):
    """Tables of more than 2^30 positions, or more than 2^31 tiles of 128 positions over all sequences and heads (pages of 16, 2 heads)."""
    c, b = cache(page_size=8 if len(kw) == 1 else 16, page_stride=1 << 12), batch(table_stride=1 << 30, **kw)
    a = _cabi.Kv4AttentionArgs(rows=2, q=P, out=P, q_stride=256, out_stride=256, q_heads=4, causal=1, scale=0.1)
    L = _cabi.lib()
    assert L.apnn_kv4_attention(None, ctypes.addressof(c), ctypes.addressof(b), ctypes.addressof(a), P, 1 << 40) == UNSUPPORTED
    assert L.apnn_kv4_attention_workspace_bytes(ctypes.addressof(c), ctypes.addressof(b), 4) == 0


def test_attention_needs_its_workspace():
    L = _cabi.lib()
    c, b = cache(), batch()
    a = _cabi.Kv4AttentionArgs(rows=2, q=P, out=P, q_stride=256, out_stride=256, q_heads=4, causal=1, scale=0.1)
    args = (None, ctypes.addressof(c), ctypes.addressof(b), ctypes.addressof(a))
    need = L.apnn_kv4_attention_workspace_bytes(ctypes.addressof(c), ctypes.addressof(b), 4)
    assert need > 0
    assert L.apnn_kv4_attention(*args, None, need) == WORKSPACE
    assert L.apnn_kv4_attention(*args, P, need - 1) == WORKSPACE
    assert L.apnn_kv4_attention(*args, P + 4, need) == ALIGNMENT
    assert L.apnn_kv4_attention_check(None, None) == INVALID


def test_python_checks():
    import apnn_tc_b200 as ap
    with pytest.raises(ValueError, match="CUDA"):
        ap.linear_planes(torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(4, 8, 4, dtype=torch.int32), torch.ones(8))
    with pytest.raises(ValueError, match="head_dim"):
        ap.KVCache4(2, 1, 16, 80)
    with pytest.raises(ValueError, match="page_size"):
        ap.KVCache4(2, 1, 24, 64)
    with pytest.raises(ValueError, match="dtype"):
        ap.KVCache4(2, 1, 16, 64, dtype=torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        ap.KVCache4(2, 1, 16, 64, data=torch.zeros(2, 1, 16 * 72 // 4, dtype=torch.int32))
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ap.KVBatch(i, i[:2], i.view(1, 3), 1)


def test_descriptors_match_the_header():
    """The structures' sizes as the C compiler lays them out."""
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"apnn_linear_desc": _cabi.LinearDesc, "apnn_kv4_cache": _cabi.Kv4Cache, "apnn_kv4_batch": _cabi.Kv4Batch,
             "apnn_kv4_append_args": _cabi.Kv4AppendArgs, "apnn_kv4_attention_args": _cabi.Kv4AttentionArgs}
    lines = []
    for n, s in names.items():
        lines += [f'printf("%zu\\n", sizeof({n}));'] + [f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in s._fields_]
    with tempfile.TemporaryDirectory() as d:
        src = os.path.join(d, "a.c")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include <stddef.h>\n#include "apnn_b200.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
        subprocess.check_call(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(root, "include"), src, "-o", os.path.join(d, "a")])
        got = [int(v) for v in subprocess.check_output([os.path.join(d, "a")]).split()]
    want = []
    for s in names.values():
        want += [ctypes.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_plain_quantiser(dtype):
    """Levels of a row stand for its elements to within half a step and the roundings of step and lowest value."""
    rng = np.random.default_rng(3)
    x = rng.normal(size=(50, 64)).astype(np.float32)
    x[0] = 1.5
    x[1, 3] = np.inf
    level, step, low = ref.quantise(x, dtype)
    assert (level[0] == 0).all() and step[0] == 0 and low[0] == 1.5
    assert np.isnan(step[1]).all() and (level[1] == 0).all()
    y = step[2:] * level[2:].astype(np.float64) + low[2:]
    e = ref.STEP[dtype]
    assert (np.abs(y - x[2:]) <= step[2:] * (0.5 + 2.0 ** -20) + e * (np.abs(low[2:]) + 16 * step[2:])).all()
