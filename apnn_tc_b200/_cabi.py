"""ctypes binding of ``libapnn_b200.so`` (the C ABI declared in ``include/apnn_b200.h``).

There is no fallback: if the shared object is missing or a call fails, an exception is
raised.  ``python -m apnn_tc_b200.build`` produces the library.
"""
from __future__ import annotations

import ctypes
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libapnn_b200.so")

# enums of include/apnn_b200.h
OUT_INT32, OUT_LOWBITS, OUT_THRESHOLDS, OUT_FLOAT = 0, 1, 2, 3
QUANT_CENTRED = 0x100   # flag in the `bits` argument of the first-layer int8 gathers
ROWS_I8, ROWS_FP4 = 1, 2   # Epilogue.out_i8: one byte, or one e2m1 nibble, per output element
SIGN_NONE, SIGN_W, SIGN_X = 0, 1, 2
POOL_NONE, POOL_AVG2, POOL_MAX2 = 0, 1, 2
ALGO_AUTO, ALGO_BMMA, ALGO_IMMA, ALGO_TCGEN05, ALGO_TCGEN05_PAIR = 0, 1, 2, 3, 4
TYPE_BF16, TYPE_FP16, TYPE_FP32 = 0, 1, 2
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
ALGOS = {"auto": ALGO_AUTO, "bmma": ALGO_BMMA, "imma": ALGO_IMMA, "tcgen05": ALGO_TCGEN05, "tcgen05_pair": ALGO_TCGEN05_PAIR}

# every symbol the header declares; the CPU test-suite checks the library exports them all
EXPORTS = (
    "apnn_status_string", "apnn_last_cuda_error", "apnn_version", "apnn_gemm", "apnn_gemm_ex",
    "apnn_gemm_workspace_bytes", "apnn_gemm_check", "apnn_expand_planes", "apnn_expand_planes_pair", "apnn_gemm_i8", "apnn_gemm_w8", "apnn_expand_planes_fp4", "apnn_gemm_fp4", "apnn_gemm_static_scratch", "apnn_conv2d", "apnn_conv2d_ex",
    "apnn_conv2d_workspace_bytes", "apnn_conv2d_check", "apnn_conv2d_i8", "apnn_bit_compress", "apnn_quantize_pack", "apnn_quantize_im2col", "apnn_create",
    "apnn_destroy", "apnn_gemm_host", "apnn_conv2d_host", "apnn_probe_peak", "apnn_quantize_im2col_i8", "apnn_quantize_window_rows_i8", "apnn_quantize_blocks_i8", "apnn_maxpool2x2_i8", "apnn_requantize_i32",
    "apnn_conv2d_fp4", "apnn_linear_fp4", "apnn_gemm_planes", "apnn_conv2d_i8_to_fp4", "apnn_maxpool2x2_rows",
    "apnn_linear_planes", "apnn_linear_planes_plan", "apnn_kv4_append", "apnn_kv4_read", "apnn_kv4_attention", "apnn_kv4_attention_workspace_bytes",
    "apnn_kv4_attention_check",
)


class Epilogue(ctypes.Structure):
    """``apnn_epilogue``; ``struct_size`` is filled in on construction (APNN_EPILOGUE_INIT)."""
    _fields_ = [
        ("struct_size", ctypes.c_uint32),
        ("out_mode", ctypes.c_int32),
        ("out_bits", ctypes.c_int32),
        ("signed_operand", ctypes.c_int32),
        ("pool", ctypes.c_int32),
        ("out_halo", ctypes.c_int32),
        ("in_halo", ctypes.c_int32),
        ("thresholds", ctypes.c_void_p),
        ("residual_in", ctypes.c_void_p),
        ("residual_out", ctypes.c_void_p),
        ("n_peer_out", ctypes.c_int32),
        ("out_i8", ctypes.c_int32),
        ("peer_out", ctypes.c_void_p * 7),
        ("residual_i16", ctypes.c_int32),
        ("affine_scale", ctypes.c_void_p),
        ("affine_bias", ctypes.c_void_p),
    ]

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.struct_size = ctypes.sizeof(Epilogue)


class _Sized(ctypes.Structure):
    """A descriptor whose first member records its size."""
    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.struct_size = ctypes.sizeof(self)


class LinearDesc(_Sized):
    """``apnn_linear_desc``"""
    _fields_ = [("struct_size", ctypes.c_uint32), ("x_type", ctypes.c_int32), ("out_type", ctypes.c_int32), ("activation", ctypes.c_int32),
                ("zero", ctypes.c_float), ("scale", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("residual", ctypes.c_void_p),
                ("ldx", ctypes.c_int64), ("ldo", ctypes.c_int64), ("ldr", ctypes.c_int64)]


class Kv4Cache(_Sized):
    """``apnn_kv4_cache``"""
    _fields_ = [("struct_size", ctypes.c_uint32), ("type", ctypes.c_int32), ("data", ctypes.c_void_p), ("page_stride", ctypes.c_int64),
                ("pages", ctypes.c_int32), ("heads", ctypes.c_int32), ("page_size", ctypes.c_int32), ("head_dim", ctypes.c_int32)]


class Kv4Batch(_Sized):
    """``apnn_kv4_batch``"""
    _fields_ = [("struct_size", ctypes.c_uint32), ("sequences", ctypes.c_int32), ("cu_q", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("table", ctypes.c_void_p), ("table_stride", ctypes.c_int64), ("table_width", ctypes.c_int32), ("max_q", ctypes.c_int32)]


class Kv4AppendArgs(_Sized):
    """``apnn_kv4_append_args``"""
    _fields_ = [("struct_size", ctypes.c_uint32), ("rows", ctypes.c_int32), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_stride", ctypes.c_int64), ("v_stride", ctypes.c_int64), ("q", ctypes.c_void_p), ("q_out", ctypes.c_void_p),
                ("q_stride", ctypes.c_int64), ("q_out_stride", ctypes.c_int64), ("q_heads", ctypes.c_int32),
                ("rotary_dim", ctypes.c_int32), ("q_norm", ctypes.c_void_p), ("k_norm", ctypes.c_void_p), ("eps", ctypes.c_double),
                ("interleaved", ctypes.c_int32), ("rotary", ctypes.c_void_p), ("rotary_rows", ctypes.c_int32)]


class Kv4AttentionArgs(_Sized):
    """``apnn_kv4_attention_args``"""
    _fields_ = [("struct_size", ctypes.c_uint32), ("rows", ctypes.c_int32), ("q", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("lse", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("out_stride", ctypes.c_int64), ("q_heads", ctypes.c_int32),
                ("causal", ctypes.c_int32), ("window", ctypes.c_int32), ("scale", ctypes.c_float)]


_FORMATS = {ctypes.c_uint32: "I", ctypes.c_int32: "i", ctypes.c_int64: "q", ctypes.c_void_p: "P", ctypes.c_float: "f", ctypes.c_double: "d"}


def packer(descriptor):
    """A function that packs a descriptor's fields (all but ``struct_size``, null pointers as 0) into bytes of its layout."""
    layout = struct.Struct("@" + "".join(_FORMATS[t] for _, t in descriptor._fields_) + "0q")
    assert layout.size == ctypes.sizeof(descriptor), descriptor
    pack, size = layout.pack, layout.size
    return lambda *fields: pack(size, *fields)


class ApnnError(RuntimeError):
    def __init__(self, status: int, text: str):
        super().__init__(text)
        self.status = status


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python -m apnn_tc_b200.build` (there is no CPU fallback)")
    L = ctypes.CDLL(LIB_PATH)
    vp, i, sz, lg = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_long
    ep = ctypes.POINTER(Epilogue)
    L.apnn_status_string.restype = ctypes.c_char_p
    L.apnn_status_string.argtypes = [i]
    L.apnn_last_cuda_error.restype = ctypes.c_char_p
    L.apnn_version.restype = i
    L.apnn_gemm.argtypes = [vp, i, i, vp, vp, vp, i, i, i]
    L.apnn_gemm_ex.argtypes = [vp, i, i, i, vp, vp, vp, i, i, i, ep, vp, sz]
    L.apnn_gemm_workspace_bytes.restype = sz
    L.apnn_gemm_workspace_bytes.argtypes = [i, i, i, i, i, i]
    L.apnn_gemm_check.argtypes = [vp, vp, i, i, i]
    L.apnn_expand_planes.argtypes = [vp, vp, vp, lg, i, i, i]
    L.apnn_expand_planes_pair.argtypes = [vp, vp, vp, lg, i, i, vp, vp, lg, i, i, i]
    L.apnn_gemm_i8.argtypes = [vp, vp, vp, vp, i, i, i, i, i, ep, vp]
    L.apnn_gemm_w8.argtypes = [vp, vp, i, vp, vp, i, i, i, i, i, ep, vp]
    L.apnn_expand_planes_fp4.argtypes = [vp, vp, vp, lg, i, i, i]
    L.apnn_gemm_fp4.argtypes = [vp, vp, vp, vp, i, i, i, ep, vp]
    L.apnn_gemm_static_scratch.argtypes = [vp, i, i, vp, vp, vp, i, i, i, ep, vp]
    L.apnn_conv2d.argtypes = [vp, i, i, vp, vp, vp, i, i, i, i, i, i, i, ep]
    L.apnn_conv2d_ex.argtypes = [vp, i, i, i, vp, vp, vp, i, i, i, i, i, i, i, ep, vp, sz]
    L.apnn_conv2d_workspace_bytes.restype = sz
    L.apnn_conv2d_workspace_bytes.argtypes = [i, i, i, i, i, i, i]
    L.apnn_conv2d_check.argtypes = [vp, vp, i, i, i, i, i, i]
    L.apnn_conv2d_i8.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, i, i, ep, vp]
    L.apnn_bit_compress.argtypes = [vp, vp, vp, lg, i, i]
    L.apnn_quantize_pack.argtypes = [vp, vp, vp, lg, i, i]
    L.apnn_probe_peak.argtypes = [vp, i, i, vp, ctypes.POINTER(ctypes.c_double)]
    L.apnn_quantize_im2col.argtypes = [vp, vp, vp, i, i, i, i, i, i, i]
    L.apnn_quantize_im2col_i8.argtypes = [vp, vp, vp, i, i, i, i, i, i, i, i]
    L.apnn_quantize_window_rows_i8.argtypes = [vp, vp, vp, i, i, i, i, i, i, i, i]
    L.apnn_quantize_blocks_i8.argtypes = [vp, vp, vp, i, i, i, i, i, i, i, i]
    L.apnn_maxpool2x2_i8.argtypes = [vp, vp, vp, i, i, i, i, i, i]
    L.apnn_conv2d_i8_to_fp4.argtypes = L.apnn_conv2d_i8.argtypes
    L.apnn_gemm_planes.argtypes = [vp, i, i, vp, vp, vp, i, i, i, ep, vp]
    L.apnn_linear_fp4.argtypes = [vp, vp, vp, vp, i, i, i, ep, vp]
    L.apnn_conv2d_fp4.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, ep, vp]
    L.apnn_maxpool2x2_rows.argtypes = [vp, vp, vp, i, i, i, i, i, i, i, i]
    L.apnn_requantize_i32.argtypes = [vp, vp, vp, ctypes.c_long, i, vp]
    L.apnn_create.argtypes = [ctypes.POINTER(vp), i]
    L.apnn_destroy.argtypes = [vp]
    L.apnn_gemm_host.argtypes = [vp, i, i, i, vp, vp, vp, i, i, i, ep]
    L.apnn_conv2d_host.argtypes = [vp, i, i, vp, vp, vp, i, i, i, i, i, i, i, ep]
    L.apnn_linear_planes.argtypes = [vp, i, vp, vp, vp, i, i, i, vp, vp]
    L.apnn_linear_planes_plan.argtypes = [i, i, i, vp, vp, vp]
    L.apnn_kv4_append.argtypes = [vp, vp, vp, vp]
    L.apnn_kv4_read.argtypes = [vp, vp, vp, vp, vp, i]
    L.apnn_kv4_attention_workspace_bytes.restype = sz
    L.apnn_kv4_attention_workspace_bytes.argtypes = [vp, vp, i]
    L.apnn_kv4_attention.argtypes = [vp, vp, vp, vp, vp, sz]
    L.apnn_kv4_attention_check.argtypes = [vp, vp]
    _lib = L
    return L


def check(status: int, what: str = "") -> None:
    if status != 0:
        L = lib()
        text = L.apnn_status_string(status).decode()
        if status == 5:
            text += ": " + L.apnn_last_cuda_error().decode()
        raise ApnnError(status, f"{what}: {text}" if what else text)
