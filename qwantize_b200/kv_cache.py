"""A paged key / value cache held in 8 bits, and attention over it.

``KVCache8`` holds pages of 64 tokens in int8 or E4M3 with one fp32 scale for each
page and head, for keys and values apart.  ``kv_cache_append`` puts new tokens
in (a prompt's or one per sequence), ``kv_cache_attention`` attends one query
token per sequence to them, ``kv_cache_read`` gives pages back as numbers.  Block
tables and lengths are the caller's, device tensors of int32 (int64 is converted on
each call, two small kernels a tensor).  None has a gradient:
inputs that require one are refused outside torch.no_grad()."""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L
from .core import cuda_device

PAGE = 64
_KV = {torch.int8: L.KV_INT8, torch.float8_e4m3fn: L.KV_E4M3}
_workspace = {}  # (device, D) -> bytes


class KVCache8(L.Bound):
    """num_pages pages of 64 tokens for kv_heads heads of head_dim (64 or 128)
    values, in dtype torch.int8 or torch.float8_e4m3fn.

    k, v: (num_pages, kv_heads, 64 * head_dim) bytes in the order the kernels
    read; k_scale, v_scale: (num_pages, kv_heads) fp32.  Can be copied, pickled and
    saved."""

    page = PAGE
    _bound = ("device", "lib", "args")

    def __init__(self, num_pages, kv_heads, head_dim, dtype=torch.int8, device="cuda"):
        assert dtype in _KV, f"dtype={dtype}, expected torch.int8 or torch.float8_e4m3fn"
        assert head_dim in (64, 128), f"head_dim={head_dim}, expected 64 or 128"
        assert torch.device(device).type == "cuda", f"device={device}, a cache lives on a CUDA device"
        assert num_pages >= 0 and 1 <= kv_heads <= 1024, "need num_pages >= 0 and 1 to 1024 kv_heads"
        if not torch.cuda.is_available():
            raise RuntimeError("qwantize_b200 needs a CUDA (sm_100a) device; none is available")
        self.num_pages, self.kv_heads, self.head_dim, self.dtype = num_pages, kv_heads, head_dim, dtype
        self.k = torch.zeros(num_pages, kv_heads, PAGE * head_dim, dtype=torch.uint8, device=device)
        self.v = torch.zeros_like(self.k)
        self.k_scale = torch.zeros(num_pages, kv_heads, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)
        self._bind()

    def _bind(self):
        self.device = dev = cuda_device(self.k)
        for name in ("k", "v", "k_scale", "v_scale"):
            setattr(self, name, getattr(self, name).to(dev))
        self.lib = L.load()
        # the pointers and sizes that every call passes on
        self.args = (self.k.data_ptr(), self.k_scale.data_ptr(), self.v.data_ptr(), self.v_scale.data_ptr(), _KV[self.dtype],
                     self.num_pages, self.kv_heads, self.head_dim)

    def load_codes(self, k, k_scale, v, v_scale):
        """Set the whole cache from codes (num_pages, kv_heads, 64, head_dim) of its
        dtype and scales (num_pages, kv_heads)."""
        P, H, D = self.num_pages, self.kv_heads, self.head_dim
        for c, s in ((k, k_scale), (v, v_scale)):
            assert tuple(c.shape) == (P, H, PAGE, D) and c.dtype == self.dtype, f"expected {self.dtype} codes {(P, H, PAGE, D)}"
            assert tuple(s.shape) == (P, H), f"expected scales {(P, H)}"
        # keys: token 16 t + 2 j + e, value 64 h + i at (j, h, t, e, i); values transposed
        kb = k.to(self.device).view(torch.uint8).reshape(P, H, 4, 8, 2, D // 64, 64).permute(0, 1, 3, 5, 2, 4, 6)
        self.k.copy_(kb.reshape(P, H, PAGE * D))
        self.v.copy_(v.to(self.device).view(torch.uint8).transpose(2, 3).reshape(P, H, PAGE * D))
        self.k_scale.copy_(k_scale)
        self.v_scale.copy_(v_scale)

    def codes(self):
        """(k, k_scale, v, v_scale) as load_codes takes them."""
        P, H, D = self.num_pages, self.kv_heads, self.head_dim
        k = self.k.reshape(P, H, 8, D // 64, 4, 2, 64).permute(0, 1, 4, 2, 5, 3, 6).reshape(P, H, PAGE, D)
        v = self.v.reshape(P, H, D, PAGE).transpose(2, 3).contiguous()
        return k.view(self.dtype), self.k_scale.clone(), v.view(self.dtype), self.v_scale.clone()


def _index(t, name, dev, ndim):
    assert t.ndim == ndim and (t.dtype == torch.int32 or t.dtype == torch.int64), f"{name} must be a {ndim}-d int32 tensor"
    assert t.device == dev, f"{name} is on {t.device}, the cache on {dev}"
    if t.dtype != torch.int32:
        t = t.clamp(-(2**31), 2**31 - 1).to(torch.int32)  # beyond 32 bits: still beyond the cache
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _table(block_table, lengths, cache):
    assert isinstance(cache, KVCache8), "cache must be a KVCache8"
    table = _index(block_table, "block_table", cache.device, 2)
    lengths = _index(lengths, "lengths", cache.device, 1)
    B, pages = table.shape
    assert lengths.shape[0] == B, f"{lengths.shape[0]} lengths for {B} rows of block_table"
    ld = table.stride(0) if B > 1 else pages
    if ld < pages:
        table, ld = table.contiguous(), pages
    return table, lengths, B, pages, ld


def _strides(x):
    """The strides of x (n, heads, D), with those of single elements, which torch
    keeps as they were cut, also through contiguous(), as in contiguous rows."""
    s0, s1, s2 = x.stride()
    n, heads, D = x.shape
    if heads <= 1 or n == 0:
        s1 = D
    return heads * D if n <= 1 else s0, s1, s2


def _rows16(x, name, shape_tail, dev):
    """x (n, heads, D) of 16 bits with contiguous, 16-byte aligned rows, and its strides."""
    assert x.ndim == 3 and x.shape[1:] == shape_tail, f"{name} is {tuple(x.shape)}, expected (n, {shape_tail[0]}, {shape_tail[1]})"
    assert x.dtype == torch.bfloat16 or x.dtype == torch.float16, f"unsupported dtype {x.dtype}, expected bfloat16 or float16"
    assert x.device == dev, f"{name} is on {x.device}, the cache on {dev}"
    s0, s1, s2 = x.stride()
    if s2 != 1 or s1 % 8 or s0 % 8 or x.data_ptr() % 16:
        s0, s1, s2 = _strides(x)
        if s2 != 1 or s1 % 8 or s0 % 8 or x.data_ptr() % 16:
            x = x.contiguous()
            if x.data_ptr() % 16:
                x = x.clone()
            s0, s1, _ = _strides(x)
    return x, s0, s1


def kv_cache_append(cache, k, v, block_table, lengths, cu_new=None, max_new=None):
    """Put new keys and values (N, kv_heads, head_dim), bf16 or fp16, behind the
    lengths[b] tokens that each sequence has.

    block_table (B, max_pages) int32 names the page of a sequence's tokens 64 i ..
    64 i + 63.  cu_new (B + 1) int32: sequence b takes tokens cu_new[b] ..
    cu_new[b + 1] - 1, at most max_new (default N); None: one token each.  A
    page's scale grows to what its new tokens need, its older codes being taken
    over to the larger scale, and slots behind the last token become zero.  A
    page must belong to one of the sequences only.  ``lengths`` stays as it is."""
    table, lengths, B, pages, ld = _table(block_table, lengths, cache)
    if k.requires_grad or v.requires_grad:
        L.no_gradient(k=k, v=v)
    tail = (cache.kv_heads, cache.head_dim)
    k, k0, k1 = _rows16(k, "k", tail, cache.device)
    v, v0, v1 = _rows16(v, "v", tail, cache.device)
    N = k.shape[0]
    assert v.shape[0] == N and v.dtype == k.dtype, "k and v must have the same number of tokens and type"
    cu = None
    if cu_new is None:
        assert N == B, f"without cu_new there is one new token per sequence: {N} tokens, {B} sequences"
        max_new = 1
    else:
        cu_new = _index(cu_new, "cu_new", cache.device, 1)
        assert cu_new.shape[0] == B + 1, f"cu_new has {cu_new.shape[0]} entries, expected {B + 1}"
        max_new = N if max_new is None else int(max_new)
        cu = cu_new.data_ptr()
    with L.on_device(cache.device) as stream:
        st = cache.lib.qz_kv_append(*cache.args, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, L.DTYPE_CODES[k.dtype], N,
                                    table.data_ptr(), ld, pages, lengths.data_ptr(), cu, max_new, B, stream)
    if st:
        L.check(st, "qz_kv_append")


def kv_cache_read(cache, pages, dtype=torch.float32):
    """The keys and values of pages (n) int32 as numbers: two (n, kv_heads, 64,
    head_dim) tensors of dtype (fp32, bf16 or fp16).  NaN for a page that the
    cache does not have."""
    assert isinstance(cache, KVCache8), "cache must be a KVCache8"
    pages = _index(pages, "pages", cache.device, 1)
    assert dtype in L.DTYPE_CODES, f"unsupported dtype {dtype}"
    n = pages.shape[0]
    shape = (n, cache.kv_heads, PAGE, cache.head_dim)
    rows = PAGE * cache.head_dim
    strides = (cache.kv_heads * rows, rows, cache.head_dim, 1)
    k, v = L.empty(shape, strides, dtype, cache.device), L.empty(shape, strides, dtype, cache.device)
    with L.on_device(cache.device) as stream:
        st = cache.lib.qz_kv_read(*cache.args, pages.data_ptr(), n, k.data_ptr(), v.data_ptr(), L.DTYPE_CODES[dtype], stream)
    if st:
        L.check(st, "qz_kv_read")
    return k, v


def kv_cache_attention(cache, q, block_table, lengths, scale=None, out=None):
    """softmax(scale q K^T) V for one query token per sequence.

    q (B, heads, head_dim) bf16 or fp16, heads a multiple of the cache's (a
    group of neighbouring query heads shares one); the first lengths[b] tokens
    behind block_table[b] are attended to (an empty sequence gives zeros); scale
    defaults to 1 / sqrt(head_dim).  Products of 16-bit operands: codes fit fp16
    exactly, probabilities are rounded to it (2^-11 of their value for bf16 results,
    2^-22 for fp16, at most 2^-40 of the largest beside that).  Softmax and sums are fp32, the result is rounded once
    to q's type."""
    table, lengths, B, pages, ld = _table(block_table, lengths, cache)
    if q.requires_grad or (out is not None and out.requires_grad):
        L.no_gradient(q=q, out=out)
    D, dev = cache.head_dim, cache.device
    assert q.ndim == 3 and q.shape[0] == B, f"q is {tuple(q.shape)}, expected ({B}, heads, {D})"
    Hq = q.shape[1]
    assert Hq >= 1 and Hq % cache.kv_heads == 0, f"{Hq} query heads are not a multiple of {cache.kv_heads} cache heads"
    q, q0, q1 = _rows16(q, "q", (Hq, D), dev)
    assert B <= 4096, f"{B} sequences, expected at most 4096"
    if out is None:
        out = L.empty((B, Hq, D), (Hq * D, D, 1), q.dtype, dev)
    else:
        assert tuple(out.shape) == (B, Hq, D) and out.dtype == q.dtype and out.device == dev and out.is_contiguous(), (
            f"out must be a contiguous {q.dtype} tensor of shape {(B, Hq, D)} on {dev}")
    with L.on_device(dev) as stream:
        n = _workspace.get((dev, D))
        if n is None:
            b = ctypes.c_int64(0)
            L.check(cache.lib.qz_kv_attention_workspace(D, ctypes.byref(b)), "qz_kv_attention_workspace")
            n = _workspace[dev, D] = b.value
        ws = L.take_scratch(n, stream)
        try:
            st = cache.lib.qz_kv_attention(*cache.args, q.data_ptr(), q0, q1, L.DTYPE_CODES[q.dtype], B, Hq, table.data_ptr(), ld,
                                           pages, lengths.data_ptr(), D**-0.5 if scale is None else float(scale),
                                           out.data_ptr(), ws, n, stream)
        finally:
            L.give_scratch(ws)
    if st:
        L.check(st, "qz_kv_attention")
    return out
