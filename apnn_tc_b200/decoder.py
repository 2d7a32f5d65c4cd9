"""Operators of a decoder layer on low-bit weights and a 4-bit key / value cache, over torch device tensors.

* ``linear_planes`` -- 16-bit float activations times weights held as bit planes (``Bit_compression`` of their levels), with
  bias, activation and residual in the epilogue;
* ``KVCache4`` / ``KVBatch`` -- a paged cache of 4-bit rows and the sequences of one call;
* ``kv4_append`` -- new rows into the cache, with the norm of each query and key head and the rotation in the same pass;
* ``kv4_read`` -- rows back out of the cache; ``kv4_attention`` -- attention over it.

The reference has no counterpart (it runs convolutional networks).  Every call goes through the C ABI on the current stream of
the tensors' device; nothing here computes on the CPU, and nothing synchronises except ``kv4_attention_check``.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _cabi

_TYPES = {torch.bfloat16: _cabi.TYPE_BF16, torch.float16: _cabi.TYPE_FP16, torch.float32: _cabi.TYPE_FP32}


def _launch(device: torch.device, what: str, call) -> None:
    """``call(stream)`` with ``device`` current, on its current stream."""
    index = device.index
    if index == torch.cuda.current_device():
        status = call(torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = call(torch._C._cuda_getCurrentRawStream(index))
    if status:
        _cabi.check(status, what)


def _same_device(device: torch.device, **tensors: Optional[torch.Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the call runs on {device}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------------------ product
def linear_planes(x: torch.Tensor, planes: torch.Tensor, scale: torch.Tensor, *, zero: float = 0.0,
                  bias: Optional[torch.Tensor] = None, activation: str = "none", residual: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                  status_flag: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(scale * (x @ (level - zero)^T) + bias) + residual``, sums in fp32, one rounding.

    x: [M, K] bfloat16 or float16, unit element stride, rows a multiple of 8 elements apart.  planes: int32
    [wbits, N, PAD128(K)/32] for 1 to 4 bits, ``Bit_compression(levels[N, K], wbits)``.  scale, bias: float32 [N].  zero: a
    multiple of 1/2 in 0..15.  activation: "none" | "relu" | "silu" | "gelu" | "gelu_tanh".  residual and out: [M, N] of x's type,
    or float32 (``out_dtype``), unit element stride; residual may be out.  M may be 0.
    """
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    if x.dim() != 2 or planes.dim() != 3:
        raise ValueError("x must be [M, K] and planes [wbits, N, K/32]")
    M, K = x.shape
    wbits, N, words = planes.shape
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("x must be bfloat16 or float16")
    if planes.dtype not in (torch.int32, torch.uint32) or not planes.is_contiguous():
        raise ValueError("planes must be contiguous 32-bit words (torch.int32)")
    if words != (K + 127) // 128 * 4:
        raise ValueError(f"planes hold rows of {words} words, K = {K} needs {(K + 127) // 128 * 4}")
    if activation not in _cabi.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_cabi.ACTIVATIONS)}")
    for name, t in (("scale", scale), ("bias", bias)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (N,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous float32 [{N}]")
    device = x.device
    _same_device(device, planes=planes, scale=scale, bias=bias, residual=residual, out=out, status_flag=status_flag)
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or x.dtype, device=device)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise ValueError("out and out_dtype disagree")
    if out.dtype not in (x.dtype, torch.float32):
        raise ValueError("out must be of x's type or float32")
    for name, t in (("out", out), ("residual", residual)):
        if t is not None and (t.shape != (M, N) or t.dtype != out.dtype or (t.stride(1) != 1 and N > 1)):
            raise ValueError(f"{name} must be [{M}, {N}] of {out.dtype} with unit element stride")
    if x.stride(1) != 1 and K > 1:
        raise ValueError("x must have unit element stride")
    if status_flag is not None and (status_flag.dtype != torch.int32 or status_flag.numel() < 1):
        raise ValueError("status_flag must be int32")
    if M == 0:
        if status_flag is not None:
            status_flag.zero_()
        return out
    d = _cabi.LinearDesc()
    d.x_type, d.out_type, d.activation = _TYPES[x.dtype], _TYPES[out.dtype], _cabi.ACTIVATIONS[activation]
    d.zero = zero
    d.scale = scale.data_ptr()
    if bias is not None:
        d.bias = bias.data_ptr()
    # a single row may carry any stride: it is never stepped over
    d.ldx, d.ldo = (x.stride(0), out.stride(0)) if M > 1 else ((K + 7) // 8 * 8, N)
    if residual is not None:
        d.residual, d.ldr = residual.data_ptr(), residual.stride(0) if M > 1 else N
    lib = _cabi.lib()
    _launch(device, "apnn_linear_planes", lambda stream: lib.apnn_linear_planes(
        stream, wbits, planes.data_ptr(), x.data_ptr(), out.data_ptr(), M, N, K, ctypes.addressof(d), _ptr(status_flag)))
    return out


# ------------------------------------------------------------------------------------------------------------ cache
class KVCache4:
    """Keys and values in 4 bits, in pages (``apnn_kv4_cache``).

    ``data`` is int32 [pages, heads, page_size * (head_dim + 8) / 4]; a given one may be a view whose pages are further apart
    (one layer of a pool).  ``dtype`` is the type of the row parameters and of q, k, v and the attention's output.  A new cache is
    not initialised: rows that were never appended hold anything, and are never used by sequences that do not reach them.
    """

    def __init__(self, pages: int, heads: int, page_size: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 device=None, data: Optional[torch.Tensor] = None):
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("dtype must be bfloat16 or float16")
        if min(pages, heads, page_size, head_dim) <= 0:
            raise ValueError("sizes must be positive")
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page_size & (page_size - 1) or not 8 <= page_size <= 1024:
            raise ValueError("page_size must be a power of two from 8 to 1024")
        words = page_size * (head_dim + 8) // 4
        if data is None:
            data = torch.empty((pages, heads, words), dtype=torch.int32, device="cuda" if device is None else device)
        if not data.is_cuda:
            raise ValueError("data must be a CUDA tensor (there is no CPU path)")
        if data.dtype != torch.int32 or data.shape != (pages, heads, words) or data.stride(2) != 1 or (heads > 1 and data.stride(1) != words):
            raise ValueError(f"data must be int32 [{pages}, {heads}, {words}] with dense pages")
        self.data, self.dtype = data, dtype
        self.pages, self.heads, self.page_size, self.head_dim = pages, heads, page_size, head_dim
        stride = data.stride(0) * 4 if pages > 1 else heads * words * 4
        self._c = _cabi.Kv4Cache(type=_TYPES[dtype], data=data.data_ptr(), page_stride=stride, pages=pages, heads=heads,
                                 page_size=page_size, head_dim=head_dim)

    @property
    def device(self) -> torch.device:
        return self.data.device


class KVBatch:
    """The sequences of one call (``apnn_kv4_batch``).

    cu_q: int32 [B + 1], rows cu_q[b] .. cu_q[b+1] - 1 belong to sequence b.  kv_len: int32 [B], lengths that count these rows.
    table: int32 [B, width], the page of every page_size positions.  max_q: at least the most rows of a sequence in this call.
    The tensors are read when the kernels run: a program may update them in place between calls or graph replays.
    """

    def __init__(self, cu_q: torch.Tensor, kv_len: torch.Tensor, table: torch.Tensor, max_q: int):
        for name, t, dims in (("cu_q", cu_q, 1), ("kv_len", kv_len, 1), ("table", table, 2)):
            if not t.is_cuda:
                raise ValueError(f"{name} must be a CUDA tensor")
            if t.dtype != torch.int32 or t.dim() != dims or (t.shape[-1] > 1 and t.stride(-1) != 1):
                raise ValueError(f"{name} must be an int32 tensor of {dims} dimension(s) with unit element stride")
            if t.device != cu_q.device:
                raise ValueError("cu_q, kv_len and table must be on one device")
        B = kv_len.shape[0]
        if B == 0 or cu_q.shape[0] != B + 1 or table.shape[0] != B or table.shape[1] == 0:
            raise ValueError("cu_q must be [B + 1], kv_len [B] and table [B, width] with B, width >= 1")
        if max_q < 1:
            raise ValueError("max_q must be positive")
        self.cu_q, self.kv_len, self.table, self.max_q = cu_q, kv_len, table, int(max_q)
        self._c = _cabi.Kv4Batch(sequences=B, cu_q=cu_q.data_ptr(), kv_len=kv_len.data_ptr(), table=table.data_ptr(),
                                 table_stride=table.stride(0) if B > 1 else table.shape[1], table_width=table.shape[1], max_q=int(max_q))


def _rows(name: str, t: torch.Tensor, heads: Optional[int], cache: KVCache4) -> int:
    """Checks [rows, heads, D] of the cache's type with dense heads; returns the row stride in elements."""
    D = cache.head_dim
    if t.dtype != cache.dtype or t.dim() != 3 or t.shape[2] != D or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {heads if heads is not None else 'heads'}, {D}] of {cache.dtype}")
    if t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != D):
        raise ValueError(f"the heads of a row of {name} must be dense")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * D


def kv4_append(cache: KVCache4, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, *, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
               eps: float = 1e-6, rotary: Optional[torch.Tensor] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
    """The batch's rows of keys and values into the cache (``apnn_kv4_append``); returns the normed, rotated queries.

    k, v: [rows, heads, D]; q: [rows, q_heads, D] or None; views of one fused projection are taken as they are.  q_norm,
    k_norm: [D] weights in the cache's type.  rotary: float32 [positions, rotary_dim], rotary_dim/2 cosines and as many sines.
    """
    device = cache.device
    _same_device(device, k=k, v=v, q=q, q_out=q_out, q_norm=q_norm, k_norm=k_norm, rotary=rotary, batch=batch.cu_q)
    a = _cabi.Kv4AppendArgs()
    a.k_stride, a.v_stride = _rows("k", k, cache.heads, cache), _rows("v", v, cache.heads, cache)
    a.rows = k.shape[0]
    if v.shape[0] != k.shape[0] or (q is not None and q.shape[0] != k.shape[0]):
        raise ValueError("q, k and v disagree on the rows")
    if q is not None:
        a.q_stride, a.q_heads = _rows("q", q, None, cache), q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
        a.q_out_stride = _rows("q_out", q_out, q.shape[1], cache)
        if q_out.shape != q.shape:
            raise ValueError("q_out must have q's shape")
        a.q, a.q_out = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None or q_norm is not None:
        raise ValueError("q_out and q_norm need q")
    a.k, a.v = k.data_ptr(), v.data_ptr()
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None:
            if t.dtype != cache.dtype or t.shape != (cache.head_dim,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous [{cache.head_dim}] of {cache.dtype}")
            setattr(a, name, t.data_ptr())
    a.eps = eps
    if rotary is not None:
        if rotary.dtype != torch.float32 or rotary.dim() != 2 or not rotary.is_contiguous() or rotary.numel() == 0:
            raise ValueError("rotary must be a contiguous float32 [positions, rotary_dim]")
        a.rotary, a.rotary_rows, a.rotary_dim = rotary.data_ptr(), rotary.shape[0], rotary.shape[1]
        a.interleaved = 1 if interleaved else 0
    if a.rows > 0:
        lib = _cabi.lib()
        _launch(device, "apnn_kv4_append", lambda stream: lib.apnn_kv4_append(
            stream, ctypes.addressof(cache._c), ctypes.addressof(batch._c), ctypes.addressof(a)))
    return q_out


def kv4_read(cache: KVCache4, batch: KVBatch, rows: Optional[int] = None, *, k_out: Optional[torch.Tensor] = None,
             v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The batch's rows back out of the cache as (keys, values) [rows, heads, D] (``apnn_kv4_read``).

    rows: how many rows the batch holds (the last entry of cu_q); needed unless k_out or v_out says so.  Rows behind the last
    sequence are left as they were in given outputs and undefined in new ones.
    """
    given = k_out if k_out is not None else v_out
    if rows is None:
        if given is None:
            raise ValueError("kv4_read needs rows, k_out or v_out")
        rows = given.shape[0]
    shape = (rows, cache.heads, cache.head_dim)
    outs = []
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is None:
            t = torch.empty(shape, dtype=cache.dtype, device=cache.device)
        elif t.shape != shape or t.dtype != cache.dtype or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [{rows}, {cache.heads}, {cache.head_dim}] of {cache.dtype}")
        outs.append(t)
    _same_device(cache.device, k_out=outs[0], v_out=outs[1], batch=batch.cu_q)
    if rows > 0:
        lib = _cabi.lib()
        _launch(cache.device, "apnn_kv4_read", lambda stream: lib.apnn_kv4_read(
            stream, ctypes.addressof(cache._c), ctypes.addressof(batch._c), outs[0].data_ptr(), outs[1].data_ptr(), rows))
    return outs[0], outs[1]


# ------------------------------------------------------------------------------------------------------------ attention
def kv4_attention_workspace_bytes(cache: KVCache4, batch: KVBatch, q_heads: int) -> int:
    """Device memory that ``kv4_attention`` needs for batches of these bounds (sequences, table width, max_q)."""
    return int(_cabi.lib().apnn_kv4_attention_workspace_bytes(ctypes.addressof(cache._c), ctypes.addressof(batch._c), q_heads))


def kv4_attention(cache: KVCache4, batch: KVBatch, q: torch.Tensor, *, scale: Optional[float] = None, causal: bool = True,
                  window: int = 0, out: Optional[torch.Tensor] = None, lse=False, workspace: Optional[torch.Tensor] = None):
    """Attention of the batch's rows over the cache (``apnn_kv4_attention``); returns out, or (out, lse) where lse is asked for.

    q: [rows, q_heads, D], q_heads a multiple of the cache's heads.  scale: 1 / sqrt(D) unless given.  window: how many
    positions back a row sees, itself included (0: all); needs causal.  lse: True, or a float32 [rows, q_heads] to write.
    workspace: ``kv4_attention_workspace_bytes`` bytes (uint8), used by one call at a time; allocated here if None.
    """
    device = cache.device
    a = _cabi.Kv4AttentionArgs()
    a.q_stride = _rows("q", q, None, cache)
    rows, q_heads, D = q.shape
    if out is None:
        out = torch.empty((rows, q_heads, D), dtype=q.dtype, device=device)
    a.out_stride = _rows("out", out, q_heads, cache)
    if out.shape != q.shape:
        raise ValueError("out must have q's shape")
    with_lse = lse is not False and lse is not None
    if lse is True:
        lse = torch.empty((rows, q_heads), dtype=torch.float32, device=device)
    if with_lse and (lse.dtype != torch.float32 or lse.shape != (rows, q_heads) or not lse.is_contiguous()):
        raise ValueError(f"lse must be a contiguous float32 [{rows}, {q_heads}]")
    if window and not causal:
        raise ValueError("a window needs causal")
    if workspace is None:
        workspace = torch.empty(max(1, kv4_attention_workspace_bytes(cache, batch, q_heads)), dtype=torch.uint8, device=device)
    _same_device(device, q=q, out=out, lse=lse if with_lse else None, workspace=workspace, batch=batch.cu_q)
    a.rows, a.q_heads = rows, q_heads
    a.q, a.out = q.data_ptr(), out.data_ptr()
    if with_lse:
        a.lse = lse.data_ptr()
    a.causal, a.window = (1 if causal else 0), window
    a.scale = 1.0 / math.sqrt(D) if scale is None else scale
    if rows > 0:
        lib = _cabi.lib()
        size = workspace.numel() * workspace.element_size()
        _launch(device, "apnn_kv4_attention", lambda stream: lib.apnn_kv4_attention(
            stream, ctypes.addressof(cache._c), ctypes.addressof(batch._c), ctypes.addressof(a), workspace.data_ptr(), size))
    return (out, lse) if with_lse else out


def kv4_attention_check(workspace: torch.Tensor) -> None:
    """Synchronise and raise if the attention that last used ``workspace`` gave up on a wait."""
    lib = _cabi.lib()
    _launch(workspace.device, "apnn_kv4_attention_check", lambda stream: lib.apnn_kv4_attention_check(stream, workspace.data_ptr()))
