"""ctypes binding of libqwantize_b200.so (the C ABI in include/qwantize_b200.h).

The library is loaded from this package directory (built in-tree by
``python -m qwantize_b200.build``).  There is no fallback: if the library or a
sm_100 GPU is missing, every entry point raises.
"""
from __future__ import annotations

import ctypes
import os

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libqwantize_b200.so")

QZ_OK, QZ_ERR_INVALID, QZ_ERR_CUDA, QZ_ERR_TIMEOUT, QZ_ERR_UNSUPPORTED = 0, 1, 2, 3, 4
DTYPE_F32, DTYPE_BF16, DTYPE_F16 = 0, 1, 2
FMT_NVFP4, FMT_MXFP4 = 0, 1
FMT_NVINT4, FMT_INT8 = 3, 4  # symmetric integer grids (nvint4/, int8/ of the reference)
METHOD_NAIVE, METHOD_SSE, METHOD_HESSIAN, METHOD_NAIVE_ARGMIN, METHOD_TWO_ARGMIN = 0, 1, 2, 3, 4
KV_INT8, KV_E4M3 = 0, 1
GRAM_FULL, GRAM_BLOCKDIAG, GRAM_FULL_UPPER_TILES = 0, 1, 2

# every symbol include/qwantize_b200.h declares
EXPORTS = [
    "qz_quantize", "qz_dequantize", "qz_dequantize_packed", "qz_fp4_unpack", "qz_gram",
    "qz_weight_error_sums", "qz_output_error_sums", "qz_scale_table", "qz_last_error",
    "qz_version", "qz_device_ok", "qz_poll_device_error", "qz_gram_full_noalloc", "qz_admm",
    "qz_quantize_table", "qz_selftest_wait", "qz_quantize_grouped", "qz_gptq", "qz_spd_inverse",
    "qz_gram_unpack", "qz_fp4_scale_layout_bytes", "qz_fp4_scale_layout", "qz_fp4_linear_workspace",
    "qz_fp4_linear", "qz_moe_layout", "qz_moe_workspace", "qz_moe", "qz_kv_append", "qz_kv_read",
    "qz_kv_attention_workspace", "qz_kv_attention",
]


class QzQuantItem(ctypes.Structure):
    """One input of qz_quantize_grouped (include/qwantize_b200.h)."""
    _fields_ = [("x", ctypes.c_void_p), ("n_blocks", ctypes.c_int64), ("scales", ctypes.c_void_p),
                ("quants", ctypes.c_void_p), ("dq", ctypes.c_void_p), ("scale_codes", ctypes.c_void_p),
                ("packed", ctypes.c_void_p), ("dq_bf16", ctypes.c_void_p)]

_lib = None


class QwantizeError(RuntimeError):
    pass


def load():
    """Load and type the library (CPU-safe: no device call happens here)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: run `python -m qwantize_b200.build` first")
    L = ctypes.CDLL(LIB_PATH)
    vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
    L.qz_quantize.argtypes = [vp, i32, i64, i32, i32, i32, vp, i64, vp, vp, vp, vp, vp, vp, vp]
    L.qz_dequantize.argtypes = [vp, vp, i64, i32, vp, vp]
    L.qz_quantize_table.argtypes = [vp, i32, i64, i32, i32, vp, i32, vp, i64, vp, vp, vp, vp, vp, vp, vp]
    L.qz_admm.argtypes = [vp, i32, i64, i32, vp, vp, vp, i64, i32, i32, ctypes.c_float, vp, vp, vp, vp, vp,
                          vp, vp]
    L.qz_dequantize_packed.argtypes = [vp, vp, i64, i32, i32, vp, vp, vp]
    L.qz_fp4_unpack.argtypes = [vp, i64, vp, vp]
    L.qz_gram.argtypes = [vp, i64, i64, i32, i32, i32, vp, vp]
    L.qz_gram_full_noalloc.argtypes = [vp, i64, i64, i32, vp, vp]
    L.qz_weight_error_sums.argtypes = [vp, i32, vp, i32, i64, vp, vp]
    L.qz_output_error_sums.argtypes = [vp, i64, i64, vp, vp, i64, vp, vp]
    L.qz_scale_table.argtypes = [i32, vp, vp]
    L.qz_poll_device_error.argtypes = [i32, vp]
    L.qz_selftest_wait.argtypes = [ctypes.c_uint64, vp]
    L.qz_quantize_grouped.argtypes = [vp, i32, i32, i32, i32, i32, vp]
    L.qz_spd_inverse.argtypes = [vp, i64, vp, vp, vp]
    L.qz_gram_unpack.argtypes = [vp, i64, vp, vp]
    L.qz_gptq.argtypes = [vp, vp, vp, vp, vp, i64, i64, i32, i32, i32, i32, vp, vp, vp]
    L.qz_fp4_scale_layout_bytes.argtypes = [i64, i64, i32, vp]
    L.qz_fp4_scale_layout.argtypes = [vp, i64, i64, i32, vp, vp]
    L.qz_fp4_linear_workspace.argtypes = [i64, i64, i64, i32, vp]
    L.qz_fp4_linear.argtypes = [vp, i32, i64, i64, i64, i64, i32, vp, i64, vp, ctypes.c_float, vp, i32, vp, i32, i64,
                                vp, i64, vp]
    f32 = ctypes.c_float
    L.qz_moe_layout.argtypes = [vp, vp, i64, i64, i64, i32, i32, vp, vp, vp, vp]
    L.qz_moe_workspace.argtypes = [i64, i64, i64, i64, i64, vp]
    L.qz_moe.argtypes = [vp, i32, i64, i64, i64, i64, i64, i64, i32, vp, i32, i32, vp, vp, vp, f32, vp, vp, f32, vp,
                         vp, vp, vp, i64, vp]
    L.qz_kv_append.argtypes = [vp, vp, vp, vp, i32, i64, i64, i64, vp, i64, i64, vp, i64, i64, i32, i64, vp, i64, i64, vp,
                               vp, i64, i64, vp]
    L.qz_kv_read.argtypes = [vp, vp, vp, vp, i32, i64, i64, i64, vp, i64, vp, vp, i32, vp]
    L.qz_kv_attention_workspace.argtypes = [i64, vp]
    L.qz_kv_attention.argtypes = [vp, vp, vp, vp, i32, i64, i64, i64, vp, i64, i64, i32, i64, i64, vp, i64, i64, vp, f32,
                                  vp, vp, i64, vp]
    for name in EXPORTS:
        getattr(L, name).restype = ctypes.c_int
    L.qz_last_error.restype = ctypes.c_char_p
    _lib = L
    return L


def check(status: int, what: str = "") -> None:
    if status == QZ_OK:
        return
    msg = load().qz_last_error().decode(errors="replace")
    if status == QZ_ERR_INVALID:
        raise AssertionError(msg)
    raise QwantizeError(f"{what}: {msg} (status {status})")


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_ptr(device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


class on_device:
    """``with on_device(dev) as stream``: dev is the current device inside, and
    stream the handle of its current stream (a decode step's calls are short enough
    that the general context manager and stream object would show)."""

    __slots__ = ("index", "previous")

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.previous = torch._C._cuda_exchangeDevice(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.previous != self.index:
            torch._C._cuda_exchangeDevice(self.previous)
        return False


# Scratch memory of one call from torch's caching allocator, on the call's stream:
# released right after the launches, it is reused only by later work of that stream.
# (A tensor would do the same at three times the host time.)
take_scratch = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_alloc", None)
give_scratch = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_delete", None)


class Bound:
    """An object that keeps what every call passes on (the library, pointers) beside
    its tensors: the attributes that ``_bind`` sets.  Copies and pickles carry the
    tensors and bind themselves again."""

    _bound = ()  # the attributes that _bind sets

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in self._bound}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._bind()


def no_gradient(**tensors):
    """Refuse what a backward pass would be expected of: the serving operators have
    none, and a result without a gradient function would drop it silently."""
    if torch.is_grad_enabled():
        for name, t in tensors.items():
            assert t is None or not t.requires_grad, (
                f"{name} requires a gradient, which this operator does not have: call it under torch.no_grad()")


def empty(shape, strides, dtype, device):
    """An uninitialised contiguous tensor: with its strides given, torch takes 1.4
    us of host time instead of 2.3."""
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


DTYPE_CODES = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.bfloat16:
        return DTYPE_BF16
    if dt == torch.float16:
        return DTYPE_F16
    if dt == torch.float32:
        return DTYPE_F32
    raise ValueError(f"unsupported dtype {dt}")


def scale_table(fmt: int) -> torch.Tensor:
    buf = (ctypes.c_float * 256)()
    n = ctypes.c_int(0)
    check(load().qz_scale_table(fmt, buf, ctypes.byref(n)), "qz_scale_table")
    return torch.tensor(list(buf)[: n.value], dtype=torch.float32)
