"""Host-side checks of the serving operators' C entry points: sizes, types and
pointers are refused with a message before any device call."""
import ctypes

import pytest
import torch

from qwantize_b200 import _lib


def refused(status, word):
    assert status == _lib.QZ_ERR_INVALID
    assert word in _lib.load().qz_last_error()
    with pytest.raises(AssertionError):
        _lib.check(status)


def test_linear_sizes():
    L = _lib.load()
    n = ctypes.c_int64(0)
    for K, fmt, word in ((8, 0, b"multiple of the block size"), (16, 1, b"multiple of the block size"), (64, 4, b"NVFP4"), (0, 0, b"K > 0")):
        refused(L.qz_fp4_scale_layout_bytes(10, K, fmt, ctypes.byref(n)), word)
        refused(L.qz_fp4_linear_workspace(3, K, 10, fmt, ctypes.byref(n)), word)
    refused(L.qz_fp4_scale_layout_bytes(10, 32, 0, None), b"NULL")
    # 10 rows pad to 256, K to 256: two row tiles of four groups of 512 bytes (MXFP4: two)
    assert L.qz_fp4_scale_layout_bytes(10, 32, _lib.FMT_NVFP4, ctypes.byref(n)) == _lib.QZ_OK and n.value == 2 * 4 * 512
    assert L.qz_fp4_scale_layout_bytes(257, 288, _lib.FMT_MXFP4, ctypes.byref(n)) == _lib.QZ_OK and n.value == 4 * 2 * 2 * 512


def test_linear_arguments():
    L = _lib.load()
    ok = dict(x=16, xd=1, ldx=64, T=2, K=64, N=4, fmt=0, w=16, ldp=32, s=16, t=1.0, b=None, bd=0, o=16, od=1, ldo=4, ws=256, n=0, st=None)

    def call(**kw):
        return L.qz_fp4_linear(*{**ok, **kw}.values())

    refused(call(x=None), b"NULL")
    refused(call(xd=7), b"dtype")
    refused(call(ldx=32), b"rows of x")
    refused(call(ldx=65), b"rows of x")
    refused(call(ldp=16), b"packed rows")
    refused(call(ldo=3), b"rows of out")
    refused(call(w=8), b"aligned")
    refused(call(ws=16), b"aligned")
    refused(call(fmt=3), b"NVFP4")
    assert call(T=0, x=None) == _lib.QZ_OK


def test_moe_arguments():
    L = _lib.load()
    n = ctypes.c_int64(0)
    for T, H, I, E, top, word in ((65, 64, 32, 4, 1, b"tokens"), (1, 48, 32, 4, 1, b"multiples of 32"), (1, 64, 16, 4, 1, b"multiples of 32"),
                                  (1, 64, 32, 513, 1, b"experts"), (1, 64, 32, 4, 5, b"top_k"), (1, 64, 32, 64, 17, b"top_k"), (1, 64, 32, 4, 0, b"top_k")):
        refused(L.qz_moe_workspace(T, H, I, E, top, ctypes.byref(n)), word)
    assert L.qz_moe_workspace(1, 64, 32, 4, 1, ctypes.byref(n)) == _lib.QZ_OK and n.value > 0
    refused(L.qz_moe_layout(16, 16, 4, 48, 64, 0, 1, 16, 16, 16, None), b"multiples of 32")
    refused(L.qz_moe_layout(16, 16, 4, 64, 64, 0, 1, 16, 16, None, None), b"NULL")
    refused(L.qz_moe(16, 0, 64, 1, 64, 32, 4, 1, 1, 16, 0, 0, 16, 16, 16, 1.0, 16, 16, 1.0, 16, None, None, 256, 1 << 20, None), b"bf16 or fp16")


def test_kv_arguments():
    L = _lib.load()
    n = ctypes.c_int64(0)
    refused(L.qz_kv_attention_workspace(96, ctypes.byref(n)), b"head dimension")
    read = lambda **kw: L.qz_kv_read(*{**dict(k=16, ks=16, v=16, vs=16, kv=0, P=4, H=2, D=64, p=16, n=1, ok=16, ov=16, dt=0, st=None), **kw}.values())  # noqa: E731
    refused(read(kv=5), b"cache type")
    refused(read(H=0), b"cache heads")
    refused(read(dt=9), b"dtype")
    refused(read(ok=8), b"aligned")
    assert read(n=0) == _lib.QZ_OK
    app = dict(k=16, ks=16, v=16, vs=16, kv=0, P=4, H=2, D=64, nk=16, k0=128, k1=64, nv=16, v0=128, v1=64, dt=1, N=2, t=16, ld=3, mp=3, ln=16,
               cu=None, mx=1, B=2, st=None)
    append = lambda **kw: L.qz_kv_append(*{**app, **kw}.values())  # noqa: E731
    refused(append(dt=0), b"bf16 or fp16")
    refused(append(N=3), b"one new token per sequence")
    refused(append(ld=2), b"max_pages")
    refused(append(k1=63), b"aligned")
    refused(append(t=None), b"NULL")
    assert append(B=0, N=0) == _lib.QZ_OK
    att = dict(k=16, ks=16, v=16, vs=16, kv=0, P=4, H=2, D=64, q=16, q0=256, q1=64, dt=1, B=2, Hq=4, t=16, ld=3, mp=3, ln=16, sc=1.0, o=16, ws=16,
               n=0, st=None)
    attend = lambda **kw: L.qz_kv_attention(*{**att, **kw}.values())  # noqa: E731
    refused(attend(Hq=5), b"multiple")
    refused(attend(B=5000), b"sequences")
    refused(attend(dt=0), b"bf16 or fp16")
    refused(attend(q1=60), b"aligned")
    refused(attend(o=None), b"NULL")
    assert attend(B=0) == _lib.QZ_OK


def test_python_refusals_without_a_device():
    import qwantize_b200 as q
    with pytest.raises(AssertionError):
        q.FP4Weight(torch.zeros(4, 2, dtype=torch.uint8), torch.zeros(4, 8, dtype=torch.uint8))
    with pytest.raises(AssertionError):
        q.FP4Weight.quantize(torch.zeros(4, 24))
    with pytest.raises(AssertionError):
        q.KVCache8(4, 2, 96)
    with pytest.raises(AssertionError):
        q.fp4_linear(torch.zeros(2, 16), None)
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError, match="CUDA"):
            q.KVCache8(4, 2, 64)
