"""Products with FP4 weights: what the quantizers of this package produce, used.

``FP4Weight`` keeps a weight in the packed NVFP4 (blocks of 16) or MXFP4 (blocks
of 32) form of ``*_quantize_packed``, with its scales in the order that the
block-scaled tensor cores read.  ``fp4_linear`` multiplies activations with it:
each row of x is quantized to the same format on the way in (qz_fp4_linear).
The reference stops at dequantized weights (nvfp4/reference.py:537-549), so
these have no counterpart there."""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L
from ._staging import to_device
from .core import cuda_device, to_host_like

BLOCK = {"nvfp4": 16, "mxfp4": 32}
_FMT = {"nvfp4": L.FMT_NVFP4, "mxfp4": L.FMT_MXFP4}
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def check_packed(scale_codes, packed, fmt):
    """(format code, N..., K, block) of a packed weight (..., N, K) in the layout
    of ``*_quantize_packed``: scale_codes (..., N, K / bs) and packed
    (..., N, K / 2) or (..., N, K / bs, bs / 2), both uint8."""
    assert fmt in _FMT, f"fmt={fmt!r}, expected one of {tuple(_FMT)}"
    bs = BLOCK[fmt]
    assert scale_codes.dtype == torch.uint8 and packed.dtype == torch.uint8, "scale_codes and packed must be uint8"
    assert scale_codes.ndim >= 2, "scale_codes must be (..., N, K / block)"
    K = scale_codes.shape[-1] * bs
    flat = (*scale_codes.shape[:-1], K // 2)
    assert tuple(packed.shape) in (flat, (*scale_codes.shape, bs // 2)), (
        f"packed {tuple(packed.shape)} does not match scale_codes {tuple(scale_codes.shape)} for {fmt} (blocks of {bs})")
    assert min(scale_codes.shape) > 0, "a packed weight must not be empty"
    assert packed.device == scale_codes.device, "scale_codes and packed must be on one device"
    return bs, K, flat


def tensor_scale_for(W, fmt):
    """The power of two that brings a weight's largest magnitude to the top of
    NVFP4's range (448 * 6); 1 for MXFP4, whose scales reach any magnitude."""
    top = float(W.abs().max()) if W.numel() else 0.0
    if fmt != "nvfp4" or not top or not math.isfinite(top):
        return 1.0
    m, e = math.frexp(top / 2688.0)
    return 2.0 ** max(-120, e - 1 if m == 0.5 else e)


def quantize_weight(W, fmt, method, X=None):
    """(scale_codes, packed, tensor_scale) of W (..., N, K) by the named method of
    the format's ``*_quantize_packed``, on the power of two of tensor_scale_for."""
    from . import mxfp4, nvfp4
    assert fmt in _FMT, f"fmt={fmt!r}, expected one of {tuple(_FMT)}"
    bs = BLOCK[fmt]
    assert W.ndim >= 2 and W.shape[-1] % bs == 0, f"the last dimension must be a multiple of {bs}"
    t = tensor_scale_for(W, fmt)
    Wb = (W / t if t != 1.0 else W).reshape(*W.shape[:-1], W.shape[-1] // bs, bs)
    fn = nvfp4.nvfp4_quantize_packed if fmt == "nvfp4" else mxfp4.mxfp4_quantize_packed
    codes, packed = fn(Wb, method=method, X=X)
    return codes, packed, t


class FP4Weight(L.Bound):
    """A weight (N, K) in packed FP4, ready for ``fp4_linear``.

    scale_codes, packed: as ``nvfp4_quantize_packed`` / ``mxfp4_quantize_packed``
    return them for W.reshape(N, K / bs, bs) (bs 16 / 32); W stands for
    tensor_scale times their value.  The codes are used where they are when
    their rows are 16-byte aligned, else copied with padded rows; the scales
    are laid out once, here.  Can be copied, pickled and saved."""

    _bound = ("device", "lib", "fmt_code", "packed_ptr", "scales_ptr", "_workspace")

    def __init__(self, scale_codes, packed, fmt="nvfp4", tensor_scale=1.0):
        self.block, self.K, flat = check_packed(scale_codes, packed, fmt)
        assert scale_codes.ndim == 2, "an FP4Weight is one matrix (N, K)"
        self.fmt, self.N, self.tensor_scale = fmt, scale_codes.shape[0], float(tensor_scale)
        dev = cuda_device(packed)
        self.scale_codes = scale_codes.to(dev).contiguous()
        p = packed.to(dev).reshape(flat).contiguous()
        self.ldp = (self.K + 31) // 32 * 16
        if self.ldp != self.K // 2 or p.data_ptr() % 16:
            padded = torch.zeros(self.N, self.ldp, dtype=torch.uint8, device=dev)
            padded[:, : self.K // 2] = p
            p = padded
        self.packed = p
        n = ctypes.c_int64(0)
        with torch.cuda.device(dev):
            L.check(L.load().qz_fp4_scale_layout_bytes(self.N, self.K, _FMT[fmt], ctypes.byref(n)), "qz_fp4_scale_layout")
            self.scales = torch.empty(n.value, dtype=torch.uint8, device=dev)
            L.check(L.load().qz_fp4_scale_layout(L.ptr(self.scale_codes), self.N, self.K, _FMT[fmt], L.ptr(self.scales),
                                                 L.stream_ptr(dev)), "qz_fp4_scale_layout")
        self._bind()

    def _bind(self):
        self.device = dev = cuda_device(self.packed)
        self.scale_codes, self.packed, self.scales = self.scale_codes.to(dev), self.packed.to(dev), self.scales.to(dev)
        self.lib, self.fmt_code = L.load(), _FMT[self.fmt]
        self.packed_ptr, self.scales_ptr = self.packed.data_ptr(), self.scales.data_ptr()
        self._workspace = {}  # tokens -> bytes

    @classmethod
    def quantize(cls, W, fmt="nvfp4", method="optimal", X=None):
        """Quantize W (N, K) by the format's "naive", "optimal" or "hessian" method
        (X: activations, for "hessian"), after division by the power of two that
        tensor_scale_for gives."""
        assert W.ndim == 2, "an FP4Weight is one matrix (N, K)"
        codes, packed, t = quantize_weight(W, fmt, method, X)
        return cls(codes, packed, fmt, t)

    def dequantize(self, dtype=torch.float32):
        """The (N, K) values the weight stands for."""
        from .core import dequantize_native
        p = self.packed[:, : self.K // 2].reshape(self.N, self.K // self.block, self.block // 2)
        v = dequantize_native(self.scale_codes, p, _FMT[self.fmt], torch.float32)
        return (v.reshape(self.N, self.K) * self.tensor_scale).to(dtype)

    def workspace_bytes(self, T):
        n = self._workspace.get(T)
        if n is None:
            b = ctypes.c_int64(0)
            L.check(L.load().qz_fp4_linear_workspace(T, self.K, self.N, _FMT[self.fmt], ctypes.byref(b)),
                    "qz_fp4_linear_workspace")
            n = self._workspace[T] = b.value
        return n


def fp4_linear(x, weight, bias=None, out_dtype=None, out=None):
    """x W^T (+ bias) for x (..., K) in bf16, fp16 or fp32 and an ``FP4Weight``.

    Each row of x is quantized to the weight's format on the way in (the naive
    rule; NVFP4 rows carry a power of two, so any magnitude fits), products and
    sums run on the block-scaled tensor cores in fp32, and the result is rounded
    once to out_dtype (default: x's).  ``out`` may supply the result's buffer, a
    contiguous (..., N) tensor.  No gradient: inputs that require one are refused
    outside torch.no_grad()."""
    assert isinstance(weight, FP4Weight), "weight must be an FP4Weight"
    dtype, codes = x.dtype, L.DTYPE_CODES
    assert dtype in codes, f"unsupported dtype {dtype}, expected one of {_DTYPES}"
    if x.requires_grad or (bias is not None and bias.requires_grad) or (out is not None and out.requires_grad):
        L.no_gradient(x=x, bias=bias, out=out)
    K, N, dev = weight.K, weight.N, weight.device
    assert x.ndim >= 1 and x.shape[-1] == K, f"x has {x.shape[-1] if x.ndim else 0} columns, the weight {K}"
    assert x.device == dev or x.device.type == "cpu", f"x is on {x.device}, the weight on {dev}"
    if out_dtype is None:
        out_dtype = dtype if out is None else out.dtype
    assert out_dtype in codes, f"unsupported dtype {out_dtype}, expected one of {_DTYPES}"
    shape = (*x.shape[:-1], N)
    xd = x if x.is_cuda else to_device(x, dev)
    if xd.ndim != 2:
        xd = xd.reshape(-1, K)
    T = xd.shape[0]
    ldx, step = xd.stride()
    if T == 1:
        ldx = K
    if step != 1 or ldx < K or ldx * xd.element_size() % 16 or xd.data_ptr() % 16:
        xd, ldx = xd.contiguous(), K
        if xd.data_ptr() % 16:
            xd = xd.clone()
    bias_ptr, bias_code = None, 0
    if bias is not None:
        assert tuple(bias.shape) == (N,) and bias.dtype in codes, f"bias must be ({N},) in one of {_DTYPES}"
        bias = bias.to(dev).contiguous()
        bias_ptr, bias_code = bias.data_ptr(), codes[bias.dtype]
    if out is None:
        y = L.empty(shape, (N, 1), out_dtype, dev) if len(shape) == 2 else torch.empty(shape, dtype=out_dtype, device=dev)
    else:
        y = out
        assert tuple(y.shape) == shape and y.dtype == out_dtype and y.device == dev and y.is_contiguous(), (
            f"out must be a contiguous {out_dtype} tensor of shape {shape} on {dev}")
    if T:
        with L.on_device(dev) as stream:
            n = weight.workspace_bytes(T)
            ws = L.take_scratch(n, stream)
            try:
                st = weight.lib.qz_fp4_linear(
                    xd.data_ptr(), codes[dtype], ldx, T, K, N, weight.fmt_code, weight.packed_ptr, weight.ldp,
                    weight.scales_ptr, weight.tensor_scale, bias_ptr, bias_code, y.data_ptr(), codes[out_dtype], N,
                    ws, n, stream)
            finally:
                L.give_scratch(ws)
        if st:
            L.check(st, "qz_fp4_linear")
    if x.is_cuda or out is not None:
        return y
    return to_host_like((y,), x.device, dev)[0]
