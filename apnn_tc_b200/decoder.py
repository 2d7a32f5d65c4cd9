"""Operators of a decoder layer on low-bit weights and a 4-bit key / value cache, over torch device tensors.

* ``linear_planes`` -- 16-bit float activations times weights held as bit planes (``Bit_compression`` of their levels), with
  bias, activation and residual in the epilogue;
* ``KVCache4`` / ``KVBatch`` -- a paged cache of 4-bit rows and the sequences of one call;
* ``kv4_append`` -- new rows into the cache, with the norm of each query and key head and the rotation in the same pass;
* ``kv4_read`` -- rows back out of the cache; ``kv4_attention`` -- attention over it.

The reference has no counterpart (it runs convolutional networks).  Every call goes through the C ABI on the current stream of
the tensors' device; nothing here computes on the CPU, and nothing synchronises except ``kv4_attention_check``.  The operators
serve: there is no backward pass, and a tensor that requires a gradient is refused outside ``torch.no_grad()``.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _cabi

_TYPES = {torch.bfloat16: _cabi.TYPE_BF16, torch.float16: _cabi.TYPE_FP16, torch.float32: _cabi.TYPE_FP32}
_INPUTS = {torch.bfloat16: _cabi.TYPE_BF16, torch.float16: _cabi.TYPE_FP16}

# The call's descriptor is packed in one go (a few hundred nanoseconds; a ctypes structure filled field by field takes several
# microseconds, as long as a small call takes on the device).
_LINEAR, _APPEND, _ATTENTION = (_cabi.packer(t) for t in (_cabi.LinearDesc, _cabi.Kv4AppendArgs, _cabi.Kv4AttentionArgs))
_get_device, _get_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _launch(index: int, what: str, fn, *args) -> None:
    """``fn(stream, *args)`` with device ``index`` current, on its current stream."""
    if index == _get_device():
        status = fn(_get_stream(index), *args)
    else:
        with torch.cuda.device(index):
            status = fn(_get_stream(index), *args)
    if status:
        _cabi.check(status, what)


def _refuse_gradient(what: str) -> None:
    if torch.is_grad_enabled():
        raise ValueError(f"{what} has no backward pass and was given a tensor that requires a gradient; call it under torch.no_grad()")


def _on(index: int, name: str, t: torch.Tensor) -> int:
    """The address of a tensor that has to lie on device ``index``."""
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, the call runs on cuda:{index}")
    return t.data_ptr()


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
    if (x.requires_grad or scale.requires_grad or (bias is not None and bias.requires_grad)
            or (residual is not None and residual.requires_grad) or (out is not None and out.requires_grad)):
        _refuse_gradient("linear_planes")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    if x.dim() != 2 or planes.dim() != 3:
        raise ValueError("x must be [M, K] and planes [wbits, N, K/32]")
    M, K = x.shape
    wbits, N, words = planes.shape
    x_dtype = x.dtype
    x_type = _INPUTS.get(x_dtype)
    if x_type is None:
        raise ValueError("x must be bfloat16 or float16")
    if planes.dtype not in (torch.int32, torch.uint32) or not planes.is_contiguous():
        raise ValueError("planes must be contiguous 32-bit words (torch.int32)")
    if words != (K + 127) // 128 * 4:
        raise ValueError(f"planes hold rows of {words} words, K = {K} needs {(K + 127) // 128 * 4}")
    act = _cabi.ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(_cabi.ACTIVATIONS)}")
    index = x.get_device()
    scale_ptr = _vector(index, "scale", scale, N)
    bias_ptr = None if bias is None else _vector(index, "bias", bias, N)
    made = out is None
    if made:
        out = x.new_empty(M, N) if out_dtype is None or out_dtype is x_dtype else x.new_empty(M, N, dtype=out_dtype)
    elif out_dtype is not None and out.dtype is not out_dtype:
        raise ValueError("out and out_dtype disagree")
    out_dtype = out.dtype
    if out_dtype is not x_dtype and out_dtype is not torch.float32:
        raise ValueError("out must be of x's type or float32")
    # a single row may carry any stride: it is never stepped over
    ldx, step = x.stride()
    if step != 1 and K > 1:
        raise ValueError("x must have unit element stride")
    ldx = ldx if M > 1 else (K + 7) // 8 * 8
    ldo = N if made else _matrix("out", out, M, N, out_dtype)
    residual_ptr, ldr = (None, 0) if residual is None else (_on(index, "residual", residual), _matrix("residual", residual, M, N, out_dtype))
    flag_ptr = None
    if status_flag is not None:
        if status_flag.dtype != torch.int32 or status_flag.numel() < 1:
            raise ValueError("status_flag must be int32")
        flag_ptr = _on(index, "status_flag", status_flag)
    if M == 0:
        if status_flag is not None:
            status_flag.zero_()
        return out
    desc = _LINEAR(x_type, _TYPES[out_dtype], act, zero, scale_ptr, bias_ptr or 0, residual_ptr or 0, ldx, ldo, ldr)
    _launch(index, "apnn_linear_planes", _cabi.lib().apnn_linear_planes, wbits, _on(index, "planes", planes), x.data_ptr(),
            _on(index, "out", out), M, N, K, desc, flag_ptr)
    return out


def _vector(index: int, name: str, t: torch.Tensor, n: int) -> int:
    if t.dtype is not torch.float32 or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [{n}]")
    return _on(index, name, t)


def _matrix(name: str, t: torch.Tensor, M: int, N: int, dtype: torch.dtype) -> int:
    """Checks [M, N] with unit element stride; returns the row stride."""
    if t.dtype is not dtype or tuple(t.shape) != (M, N):
        raise ValueError(f"{name} must be [{M}, {N}] of {dtype}")
    rows, step = t.stride()
    if step != 1 and N > 1:
        raise ValueError(f"{name} must have unit element stride")
    return rows if M > 1 else N


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
        self._index = data.get_device()
        self._like = torch.empty(0, dtype=dtype, device=data.device)      # what kv4_read's outputs are made from
        self._c = _cabi.Kv4Cache(type=_TYPES[dtype], data=data.data_ptr(), page_stride=stride, pages=pages, heads=heads,
                                 page_size=page_size, head_dim=head_dim)
        self._ptr = ctypes.addressof(self._c)

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
        self._index = cu_q.get_device()
        self._c = _cabi.Kv4Batch(sequences=B, cu_q=cu_q.data_ptr(), kv_len=kv_len.data_ptr(), table=table.data_ptr(),
                                 table_stride=table.stride(0) if B > 1 else table.shape[1], table_width=table.shape[1], max_q=int(max_q))
        self._ptr = ctypes.addressof(self._c)


def _rows(name: str, t: torch.Tensor, cache: KVCache4) -> Tuple[int, int, int]:
    """Checks [rows, heads, D] of the cache's type with dense heads; returns rows, heads and the row stride in elements."""
    D = cache.head_dim
    if t.dtype is not cache.dtype or t.dim() != 3:
        raise ValueError(f"{name} must be [rows, heads, {D}] of {cache.dtype}")
    rows, heads, d = t.shape
    row, head, step = t.stride()
    if d != D:
        raise ValueError(f"{name} must be [rows, heads, {D}] of {cache.dtype}")
    if step != 1 or (head != D and heads > 1):
        raise ValueError(f"the heads of a row of {name} must be dense")
    return rows, heads, row if rows > 1 else heads * D


def _same(cache: KVCache4, batch: KVBatch) -> int:
    if batch._index != cache._index:
        raise ValueError(f"the batch is on cuda:{batch._index}, the cache on cuda:{cache._index}")
    return cache._index


def _gain(index: int, name: str, t: torch.Tensor, cache: KVCache4) -> int:
    if t.dtype is not cache.dtype or t.dim() != 1 or t.numel() != cache.head_dim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [{cache.head_dim}] of {cache.dtype}")
    return _on(index, name, t)


def kv4_append(cache: KVCache4, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, *, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
               eps: float = 1e-6, rotary: Optional[torch.Tensor] = None, interleaved: bool = False) -> Optional[torch.Tensor]:
    """The batch's rows of keys and values into the cache (``apnn_kv4_append``); returns the normed, rotated queries.

    k, v: [rows, heads, D]; q: [rows, q_heads, D] or None; views of one fused projection are taken as they are.  q_norm,
    k_norm: [D] weights in the cache's type.  rotary: float32 [positions, rotary_dim], rotary_dim/2 cosines and as many sines.
    """
    if (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad) or (q_out is not None and q_out.requires_grad)
            or (q_norm is not None and q_norm.requires_grad) or (k_norm is not None and k_norm.requires_grad)
            or (rotary is not None and rotary.requires_grad)):
        _refuse_gradient("kv4_append")
    index = _same(cache, batch)
    rows, heads, k_stride = _rows("k", k, cache)
    v_rows, v_heads, v_stride = _rows("v", v, cache)
    if heads != cache.heads or v_heads != heads:
        raise ValueError(f"k and v must have the cache's {cache.heads} heads")
    q_ptr = q_out_ptr = q_stride = q_out_stride = q_heads = q_rows = 0
    if q is not None:
        q_rows, q_heads, q_stride = _rows("q", q, cache)
        if q_out is None:
            q_out, q_out_stride = q.new_empty(q_rows, q_heads, cache.head_dim), q_heads * cache.head_dim
        else:
            out_rows, out_heads, q_out_stride = _rows("q_out", q_out, cache)
            if out_rows != q_rows or out_heads != q_heads:
                raise ValueError("q_out must have q's shape")
        q_ptr, q_out_ptr = _on(index, "q", q), _on(index, "q_out", q_out)
    elif q_out is not None or q_norm is not None:
        raise ValueError("q_out and q_norm need q")
    if v_rows != rows or (q is not None and q_rows != rows):
        raise ValueError("q, k and v disagree on the rows")
    q_norm_ptr = 0 if q_norm is None else _gain(index, "q_norm", q_norm, cache)
    k_norm_ptr = 0 if k_norm is None else _gain(index, "k_norm", k_norm, cache)
    rotary_ptr = rotary_rows = rotary_dim = 0
    if rotary is not None:
        if rotary.dtype is not torch.float32 or rotary.dim() != 2 or not rotary.is_contiguous() or rotary.numel() == 0:
            raise ValueError("rotary must be a contiguous float32 [positions, rotary_dim]")
        rotary_rows, rotary_dim = rotary.shape
        rotary_ptr = _on(index, "rotary", rotary)
    if rows > 0:
        args = _APPEND(rows, _on(index, "k", k), _on(index, "v", v), k_stride, v_stride, q_ptr, q_out_ptr, q_stride, q_out_stride,
                       q_heads, rotary_dim, q_norm_ptr, k_norm_ptr, eps, 1 if interleaved and rotary is not None else 0, rotary_ptr, rotary_rows)
        _launch(index, "apnn_kv4_append", _cabi.lib().apnn_kv4_append, cache._ptr, batch._ptr, args)
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
    index = _same(cache, batch)
    shape = (rows, cache.heads, cache.head_dim)
    if given is not None:
        for name, t in (("k_out", k_out), ("v_out", v_out)):
            if t is not None and (t.dtype is not cache.dtype or tuple(t.shape) != shape or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous [{rows}, {cache.heads}, {cache.head_dim}] of {cache.dtype}")
    if k_out is None:
        k_out = cache._like.new_empty(*shape)
    if v_out is None:
        v_out = torch.empty_like(k_out)
    if rows > 0:
        _launch(index, "apnn_kv4_read", _cabi.lib().apnn_kv4_read, cache._ptr, batch._ptr, _on(index, "k_out", k_out),
                _on(index, "v_out", v_out), rows)
    return k_out, v_out


# ------------------------------------------------------------------------------------------------------------ attention
def kv4_attention_workspace_bytes(cache: KVCache4, batch: KVBatch, q_heads: int) -> int:
    """Device memory that ``kv4_attention`` needs for batches of these bounds (sequences, table width, max_q)."""
    return int(_cabi.lib().apnn_kv4_attention_workspace_bytes(cache._ptr, batch._ptr, q_heads))


def kv4_attention(cache: KVCache4, batch: KVBatch, q: torch.Tensor, *, scale: Optional[float] = None, causal: bool = True,
                  window: int = 0, out: Optional[torch.Tensor] = None, lse=False, workspace: Optional[torch.Tensor] = None):
    """Attention of the batch's rows over the cache (``apnn_kv4_attention``); returns out, or (out, lse) where lse is asked for.

    q: [rows, q_heads, D], q_heads a multiple of the cache's heads.  scale: 1 / sqrt(D) unless given.  window: how many
    positions back a row sees, itself included (0: all); needs causal.  lse: True, or a float32 [rows, q_heads] to write.
    workspace: ``kv4_attention_workspace_bytes`` bytes (uint8), used by one call at a time; allocated here if None.
    """
    if q.requires_grad or (out is not None and out.requires_grad):
        _refuse_gradient("kv4_attention")
    index = _same(cache, batch)
    rows, q_heads, q_stride = _rows("q", q, cache)
    if out is None:
        out_stride = q_heads * cache.head_dim
        out = torch.empty_like(q) if q_stride == out_stride else q.new_empty(rows, q_heads, cache.head_dim)
    else:
        out_rows, out_heads, out_stride = _rows("out", out, cache)
        if out_rows != rows or out_heads != q_heads:
            raise ValueError("out must have q's shape")
    with_lse = lse is not False and lse is not None
    lse_ptr = 0
    if with_lse:
        if lse is True:
            lse = torch.empty((rows, q_heads), dtype=torch.float32, device=q.device)
        if lse.dtype is not torch.float32 or tuple(lse.shape) != (rows, q_heads) or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous float32 [{rows}, {q_heads}]")
        lse_ptr = _on(index, "lse", lse)
    if window:
        if not causal:
            raise ValueError("a window needs causal")
        if window >= 1 << 31:
            raise ValueError("window must be below 2^31")
    q_ptr = _on(index, "q", q)
    if workspace is not None:
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
    else:
        workspace = torch.empty(max(1, kv4_attention_workspace_bytes(cache, batch, q_heads)), dtype=torch.uint8, device=q.device)
    if rows > 0:
        args = _ATTENTION(rows, q_ptr, _on(index, "out", out), lse_ptr, q_stride, out_stride, q_heads, 1 if causal else 0, window,
                          cache.head_dim ** -0.5 if scale is None else scale)
        _launch(index, "apnn_kv4_attention", _cabi.lib().apnn_kv4_attention, cache._ptr, batch._ptr, args,
                _on(index, "workspace", workspace), workspace.numel() * workspace.element_size())
    return (out, lse) if with_lse else out


def kv4_attention_check(workspace: torch.Tensor) -> None:
    """Synchronise and raise if the attention that last used ``workspace`` gave up on a wait."""
    if not workspace.is_cuda:
        raise ValueError("workspace must be a CUDA tensor")
    _launch(workspace.get_device(), "apnn_kv4_attention_check", _cabi.lib().apnn_kv4_attention_check, workspace.data_ptr())
