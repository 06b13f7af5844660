"""Calls of the serving operators at the edges of what they take."""
import copy
import io
import pickle

import pytest
import torch

from tests.test_gpu_kv_cache import CACHES, check, queries, setup
from tests.test_gpu_moe import make, router_of, tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_moe_into_a_view_at_an_odd_offset(dtype):
    """The kernel stores four values at once; a contiguous out of any address gets the same bits."""
    import qwantize_b200 as q
    up, down, t = make(4, 64, 32, "nvfp4", 1)
    ex = q.FP4Experts(up, down, tensor_scales=(t, t))
    r, x = router_of(4, 64, torch.bfloat16, 2), tokens(3, 64, dtype, 3)
    want = q.fp4_moe(x, r, ex, 2)
    for off in (1, 2, 3, 4):
        buf = torch.full((off + x.numel() + 5,), 7.0, dtype=dtype, device=DEV)
        out = buf[off: off + x.numel()].view(x.shape)
        assert q.fp4_moe(x, r, ex, 2, out=out) is out
        assert torch.equal(out, want) and bool((buf[:off] == 7).all()) and bool((buf[off + x.numel():] == 7).all())
        got, ids, _ = q.fp4_moe(x, r, ex, 2, return_routing=True, out=out)
        assert got is out and ids.shape == (3, 2)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("extra", [0, 130])
def test_attention_lengths_up_to_the_largest_int32(dtype, extra):
    """A length beyond the table means all of it, up to 2^31 - 1 (rounding it up to
    whole pages must not wrap); extra columns take the form of wide tables."""
    import qwantize_b200 as q
    c, codes, table, _ = setup(3, [128] * 3, 2, 64, dtype, 41)
    full = torch.cat([table, table.new_full((3, extra), -1)], 1)
    x = queries(3, 8, 64, torch.bfloat16, 42)
    have = torch.tensor([128, 70, 128], dtype=torch.int32, device=DEV)
    for big in (2**31 - 1, 2**31 - 2, 2**31 - 63, 2**31 - 64, 2**31 - 65):
        lengths = torch.tensor([big, 70, big], dtype=torch.int32, device=DEV)
        check(q.kv_cache_attention(c, x, full, lengths), x, *codes, table, have)


def test_append_takes_any_upper_limit():
    """max_new is an upper limit: one beyond the new tokens, up to 2^63 - 1, changes nothing."""
    import qwantize_b200 as q
    g = torch.Generator().manual_seed(43)
    k = torch.randn(70, 2, 64, generator=g).to(torch.bfloat16).to(DEV)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([3, 0], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 69, 70], dtype=torch.int32, device=DEV)
    caches = []
    for most in (69, None, 1 << 40, 2**63 - 1):
        caches.append(q.KVCache8(4, 2, 64))
        q.kv_cache_append(caches[-1], k, k, table, lengths, cu_new=cu, max_new=most)
    assert caches[0].k[1].any()
    assert all(torch.equal(c.k, caches[0].k) and torch.equal(c.v_scale, caches[0].v_scale) for c in caches[1:])


def test_one_sequence_of_one_head_cut_from_odd_rows():
    import qwantize_b200 as q
    c, codes, table, lengths = setup(1, [100], 1, 64, torch.int8, 44)
    wide = queries(2, 1, 68, torch.bfloat16, 45)
    for first in (0, 4):
        x = wide[:1, :, first: first + 64]
        check(q.kv_cache_attention(c, x, table, lengths), x, *codes, table, lengths)
        a, b = q.KVCache8(2, 1, 64), q.KVCache8(2, 1, 64)
        n = torch.zeros(1, dtype=torch.int32, device=DEV)
        t = torch.ones(1, 1, dtype=torch.int32, device=DEV)
        q.kv_cache_append(a, x, x, t, n)
        q.kv_cache_append(b, x.clone(), x.clone(), t, n)
        assert a.k.any() and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)


def test_gradients_are_refused_not_dropped():
    import qwantize_b200 as q
    up, down, t = make(4, 64, 32, "nvfp4", 46)
    ex, w = q.FP4Experts(up, down), q.FP4Weight(up[0][0], up[1][0])
    r, x, b = router_of(4, 64, torch.bfloat16, 47), tokens(2, 64, torch.bfloat16, 48), torch.ones(64, device=DEV)
    c, _, table, n = setup(2, [5, 6], 1, 64, torch.int8, 49)
    kv = x.reshape(2, 1, 64)
    need = lambda v: v.clone().requires_grad_()  # noqa: E731
    for call in (lambda f: q.fp4_linear(f(x), w), lambda f: q.fp4_linear(x, w, bias=f(b)), lambda f: q.fp4_moe(f(x), r, ex, 2),
                 lambda f: q.fp4_moe(x, f(r), ex, 2), lambda f: q.kv_cache_attention(c, f(kv), table, n),
                 lambda f: q.kv_cache_append(c, f(kv), kv, table, n), lambda f: q.kv_cache_append(c, kv, f(kv), table, n)):
        with pytest.raises(AssertionError, match="no_grad"):
            call(need)
        want = call(lambda v: v)
        with torch.no_grad():
            got = call(need)
        assert want is None or torch.equal(want, got)
        call(lambda v: need(v).detach())


def saved(obj, where):
    f = io.BytesIO()
    torch.save(obj, f)
    f.seek(0)
    return torch.load(f, weights_only=False, map_location=where)


@pytest.mark.parametrize("keep", [copy.copy, copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o)), lambda o: saved(o, None), lambda o: saved(o, "cpu")],
                         ids=["copy", "deepcopy", "pickle", "save", "save to cpu"])
def test_weights_experts_and_caches_can_be_kept(keep):
    import qwantize_b200 as q
    up, down, t = make(4, 64, 32, "nvfp4", 50)
    r, x = router_of(4, 64, torch.bfloat16, 51), tokens(5, 64, torch.bfloat16, 52)
    ex, w = q.FP4Experts(up, down, tensor_scales=(t, t)), q.FP4Weight(up[0][1], up[1][1], tensor_scale=t)
    odd = q.FP4Weight(down[0][0][:, :1], down[1][0][:, :1])  # K = 16: padded rows
    c, _, table, n = setup(2, [5, 70], 1, 64, torch.float8_e4m3fn, 53)
    kv = tokens(2, 64, torch.bfloat16, 54).reshape(2, 1, 64)
    for obj, call in ((w, lambda o: q.fp4_linear(x, o)), (odd, lambda o: q.fp4_linear(x[:, :16], o)), (w, lambda o: o.dequantize()),
                      (ex, lambda o: q.fp4_moe(x, r, o, 2)), (c, lambda o: q.kv_cache_attention(o, kv, table, n))):
        want = call(obj)
        other = keep(obj)
        assert torch.equal(call(other), want) and torch.equal(call(obj), want)
    # a copy is its own, but for the shallow one
    other = keep(c)
    before = c.k.clone()
    q.kv_cache_append(other, kv, kv, table, n)
    assert torch.equal(c.k, before) == (keep is not copy.copy) and not torch.equal(other.k, before)
