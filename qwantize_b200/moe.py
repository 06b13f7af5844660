"""Mixture-of-experts layers on FP4 weights, for the few tokens of a decode step.

``FP4Experts`` keeps the gated experts of one layer in the packed form of
``*_quantize_packed``, laid out once for ``fp4_moe``, which runs the whole layer:
router, top-k, gate / up, activation, down, weighted sum (qz_moe)."""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L
from ._staging import to_device
from .core import cuda_device, to_host_like
from .linear import _FMT, check_packed, quantize_weight

MAX_TOKENS = 64


def _lay_out(codes, packed, fmt, gate_up, dev):
    bs, K, flat = check_packed(codes, packed, fmt)
    assert codes.ndim == 3, "experts' weights are (E, rows, K)"
    E, rows = codes.shape[:2]
    assert rows % 32 == 0 and K % 32 == 0, f"rows ({rows}) and columns ({K}) of an expert must be multiples of 32"
    codes, packed = codes.to(dev).contiguous(), packed.to(dev).reshape(flat).contiguous()
    Kp = (K + 63) // 64 * 64
    c = torch.empty(E * rows * Kp // 2, dtype=torch.uint8, device=dev)
    s = torch.empty(E * rows * Kp // bs, dtype=torch.uint8, device=dev)
    norms = torch.empty(E, 2, dtype=torch.float32, device=dev) if gate_up else None
    with torch.cuda.device(dev):
        L.check(L.load().qz_moe_layout(L.ptr(codes), L.ptr(packed), E, rows, K, _FMT[fmt], int(gate_up), L.ptr(c),
                                       L.ptr(s), L.ptr(norms), L.stream_ptr(dev)), "qz_moe_layout")
    return c, s, norms, E, rows, K


class FP4Experts(L.Bound):
    """The experts of one layer: E gated feed-forward blocks in packed FP4.

    gate_up, down: (scale_codes, packed) as ``*_quantize_packed`` return them for
    weights (E, 2 I, H) -- the I gate rows, then the I up rows -- and (E, H, I);
    the weights stand for tensor_scales times their values.  H and I are
    multiples of 32.  Laid out once, here; the inputs are not kept.  Can be copied,
    pickled and saved."""

    _bound = ("device", "lib", "weight_args", "_workspace")

    def __init__(self, gate_up, down, fmt="nvfp4", tensor_scales=(1.0, 1.0)):
        dev = cuda_device(gate_up[0])
        self.up_codes, self.up_scales, self.up_norms, self.E, rows, self.H = _lay_out(*gate_up, fmt, True, dev)
        self.down_codes, self.down_scales, _, E, H, self.I = _lay_out(*down, fmt, False, dev)
        assert (E, H, 2 * self.I) == (self.E, self.H, rows), (
            f"gate_up ({self.E}, {rows}, {self.H}) and down ({E}, {H}, {self.I}) do not belong together")
        assert self.E <= 512, f"{self.E} experts, expected at most 512"
        self.fmt = fmt
        self.tensor_scales = float(tensor_scales[0]), float(tensor_scales[1])
        self._bind()

    def _bind(self):
        self.device = dev = cuda_device(self.up_codes)
        for name in ("up_codes", "up_scales", "up_norms", "down_codes", "down_scales"):
            setattr(self, name, getattr(self, name).to(dev))
        self.lib = L.load()
        self.weight_args = (_FMT[self.fmt], self.up_codes.data_ptr(), self.up_scales.data_ptr(), self.up_norms.data_ptr(),
                            self.tensor_scales[0], self.down_codes.data_ptr(), self.down_scales.data_ptr(),
                            self.tensor_scales[1])
        self._workspace = {}

    @classmethod
    def quantize(cls, gate_up, down, fmt="nvfp4", method="optimal"):
        """Quantize weights (E, 2 I, H) and (E, H, I) by the format's "naive" or
        "optimal" method, each after division by one power of two."""
        assert gate_up.ndim == 3 and down.ndim == 3, "experts' weights are (E, rows, K)"
        a, b = quantize_weight(gate_up, fmt, method), quantize_weight(down, fmt, method)
        return cls(a[:2], b[:2], fmt, (a[2], b[2]))

    def workspace_bytes(self, T, top_k):
        n = self._workspace.get((T, top_k))
        if n is None:
            b = ctypes.c_int64(0)
            L.check(L.load().qz_moe_workspace(T, self.H, self.I, self.E, top_k, ctypes.byref(b)), "qz_moe_workspace")
            n = self._workspace[T, top_k] = b.value
        return n


def fp4_moe(x, router_weight, experts, top_k, renormalize=True, return_routing=False, out=None):
    """The whole layer for x (..., H), at most 64 tokens, bf16 or fp16.

    Logits x router_weight^T ((E, H), fp32 or 16-bit) and their softmax are
    fp32; a token goes to the top_k largest (ties: the lowest index), weighted by
    the softmax over those (renormalize=True) or over all experts.  The
    activations stay in 16 bits, sums in fp32, the result is rounded once to x's
    type.  With return_routing: (out, ids int32 (..., top_k), weights fp32).  No
    gradient: inputs that require one are refused outside torch.no_grad()."""
    assert isinstance(experts, FP4Experts), "experts must be an FP4Experts"
    dev, H, E = experts.device, experts.H, experts.E
    dtype, codes = x.dtype, L.DTYPE_CODES
    assert dtype == torch.bfloat16 or dtype == torch.float16, f"unsupported dtype {dtype}, expected bfloat16 or float16"
    assert x.ndim >= 1 and x.shape[-1] == H, f"x has {x.shape[-1] if x.ndim else 0} columns, the experts {H}"
    assert x.device == dev or x.device.type == "cpu", f"x is on {x.device}, the experts on {dev}"
    r = router_weight
    if x.requires_grad or r.requires_grad or (out is not None and out.requires_grad):
        L.no_gradient(x=x, router_weight=r, out=out)
    assert tuple(r.shape) == (E, H), f"router_weight {tuple(r.shape)}, expected {(E, H)}"
    assert r.dtype in codes, f"unsupported dtype {r.dtype}"
    top_k = int(top_k)
    assert 1 <= top_k <= min(16, E), f"top_k={top_k}, expected 1 to {min(16, E)}"
    xd = x if x.is_cuda else to_device(x, dev)
    if xd.ndim != 2:
        xd = xd.reshape(-1, H)
    T = xd.shape[0]
    assert T <= MAX_TOKENS, f"{T} tokens, expected at most {MAX_TOKENS}"
    ldx, step = xd.stride()
    if T == 1:
        ldx = H
    if step != 1 or ldx < H or ldx % 8 or xd.data_ptr() % 16:
        xd, ldx = xd.contiguous(), H
        if xd.data_ptr() % 16:
            xd = xd.clone()
    if r.device != dev or not r.is_contiguous():
        r = r.to(dev).contiguous()
    if r.data_ptr() % 16:
        r = r.clone()
    if out is None:
        y = L.empty(x.shape, (H, 1), dtype, dev) if x.ndim == 2 else torch.empty(x.shape, dtype=dtype, device=dev)
    else:
        y = out
        assert y.shape == x.shape and y.dtype == dtype and y.device == dev and y.is_contiguous(), (
            f"out must be a contiguous {dtype} tensor of shape {tuple(x.shape)} on {dev}")
        if y.data_ptr() % 8:  # a view at an odd offset: the kernel stores four values at once
            y = torch.empty(x.shape, dtype=dtype, device=dev)
    ids = weights = None
    if return_routing:
        ids = L.empty((T, top_k), (top_k, 1), torch.int32, dev)
        weights = L.empty((T, top_k), (top_k, 1), torch.float32, dev)
        if x.ndim != 2:
            ids, weights = ids.view(*x.shape[:-1], top_k), weights.view(*x.shape[:-1], top_k)
    if T:
        n = experts.workspace_bytes(T, top_k)
        with L.on_device(dev) as stream:
            ws = L.take_scratch(n, stream)
            try:
                st = experts.lib.qz_moe(
                    xd.data_ptr(), codes[dtype], ldx, T, H, experts.I, E, top_k, 1 if renormalize else 0, r.data_ptr(),
                    codes[r.dtype], *experts.weight_args, y.data_ptr(), ids.data_ptr() if return_routing else None,
                    weights.data_ptr() if return_routing else None, ws, n, stream)
            finally:
                L.give_scratch(ws)
        if st:
            L.check(st, "qz_moe")
    if out is not None and y is not out:
        y = out.copy_(y)
    res = (y, ids, weights) if return_routing else (y,)
    if not x.is_cuda and out is None:
        res = to_host_like(res, x.device, dev)
    return res if return_routing else res[0]
