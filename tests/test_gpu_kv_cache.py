"""The 8-bit KV cache against its definition in 64 bits.

append: codes and scales are whole operations of fp32 (a maximum, divisions,
roundings) and have to equal the oracle's, which does them in numpy-like steps
with torch on the CPU.  attention, with u = 2^-24: the products of codes and fp16 rows
are exact, a score is within D 2u sum |q k| (plus 4u of it for the scales) of
its value; probabilities follow by e^(2 max error) - 1, are rounded to fp16
(2^-11, or 2^-25 of the largest) and summed in fp32 (n 2u); the output is
rounded once (2^-8 bf16, 2^-11 fp16)."""
import pytest
import torch

from tests.test_gpu_linear import ROUND

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
CACHES = [torch.int8, torch.float8_e4m3fn]


def encode(y, dtype):
    return y.round().clamp(-127, 127).to(torch.int8) if dtype == torch.int8 else y.clamp(-448, 448).to(dtype)


def fill(P, H, D, dtype, seed):
    """A cache with every page full of random codes, and the codes."""
    import qwantize_b200 as q
    g = torch.Generator().manual_seed(seed)
    mk = lambda: encode(torch.randn(P, H, 64, D, generator=g) * (40 if dtype == torch.int8 else 100), dtype)  # noqa: E731
    k, v = mk(), mk()
    ks, vs = (torch.exp(torch.randn(P, H, generator=g)) / 100 for _ in range(2))
    c = q.KVCache8(P, H, D, dtype)
    c.load_codes(k, ks, v, vs)
    return c, k, ks, v, vs


def oracle(q, k, ks, v, vs, table, lengths, scale):
    B, Hq, D = q.shape
    q = q.cpu().double()
    H = k.shape[1]
    out, lim = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64)
    for b in range(B):
        n = min(int(lengths[b]), 64 * table.shape[1])
        if n <= 0:
            continue
        pages = table[b, : -(-n // 64)].long()
        kk = (k[pages].double() * ks[pages].double()[..., None, None]).transpose(0, 1).reshape(H, -1, D)[:, :n]
        vv = (v[pages].double() * vs[pages].double()[..., None, None]).transpose(0, 1).reshape(H, -1, D)[:, :n]
        qq = q[b].reshape(H, Hq // H, D)
        s = qq @ kk.transpose(1, 2) * scale
        es = scale * D * 2 * U * (qq.abs() @ kk.abs().transpose(1, 2)) + 4 * U * s.abs()
        # the exponent is formed in base 2 from the rounded score: a few more units of its magnitude
        es = es + 4 * U * (s - s.amax(-1, keepdim=True)).abs()
        p = torch.softmax(s, -1)
        rel = torch.expm1(2 * es.amax(-1, keepdim=True)) + 2.0**-11 + 2 * U * n + 8 * U
        out[b] = (p @ vv).reshape(Hq, D)
        lim[b] = (rel * (p @ vv.abs()) + 2.0**-25 * p.amax(-1, keepdim=True) * vv.abs().sum(1, keepdim=True)).reshape(Hq, D)
    return out, lim


def check(out, q, k, ks, v, vs, table, lengths, scale=None):
    D = q.shape[2]
    ref, lim = oracle(q, k, ks, v, vs, table.cpu(), lengths.cpu(), D**-0.5 if scale is None else scale)
    lim = lim + ROUND[out.dtype] * (ref.abs() + lim) + (2.0**-25 if out.dtype == torch.float16 else 1e-30)
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= lim).all()), (float((err / lim).max()), int((err > lim).sum()))


def setup(B, lens, H, D, dtype, seed, extra=0):
    pages = max(1, max(-(-n // 64) for n in lens)) + extra
    c, *codes = fill(B * pages + 3, H, D, dtype, seed)
    g = torch.Generator().manual_seed(seed + 1)
    table = torch.randperm(B * pages + 3, generator=g)[: B * pages].int().reshape(B, pages).to(DEV)
    return c, codes, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def queries(B, Hq, D, dtype, seed):
    return (2 * torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(seed))).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,G", [
    ([1], 1, 1), ([63], 2, 4), ([64], 1, 8), ([65], 3, 5), ([300], 8, 4), ([0, 1, 2], 2, 16), ([0], 1, 2), ([0, 0, 0], 2, 2),
    ([64, 0, 128, 129, 0], 4, 1), ([5000], 2, 8), ([1000, 1, 0, 77, 640], 8, 7), ([130, 200], 1, 40), ([17] * 90, 2, 3)])
def test_attention_shapes(dtype, D, lens, H, G):
    import qwantize_b200 as q
    c, codes, table, lengths = setup(len(lens), lens, H, D, dtype, len(lens) + H + G, extra=1)
    for t in (torch.bfloat16, torch.float16):
        x = queries(len(lens), H * G, D, t, 3)
        check(q.kv_cache_attention(c, x, table, lengths), x, *codes, table, lengths)


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,H,G", [([300], 2, 1), ([1, 0, 64, 65], 3, 5), ([2000, 7, 640], 2, 8), ([1500], 1, 16), ([0], 1, 3)])
def test_narrow_and_wide_tables(dtype, D, lens, H, G):
    """A table of a few pages gives a pair of sequence and head to one CTA, a wide
    one cuts all pages evenly; the columns behind a sequence are not read."""
    import qwantize_b200 as q
    c, codes, table, lengths = setup(len(lens), lens, H, D, dtype, len(lens) + G)
    wide = torch.cat([table, table.new_full((len(lens), 130), 1 << 30)], 1)
    for t in (torch.bfloat16, torch.float16):
        x = queries(len(lens), H * G, D, t, 4)
        check(q.kv_cache_attention(c, x, table, lengths), x, *codes, table, lengths)
        check(q.kv_cache_attention(c, x, wide, lengths), x, *codes, table, lengths)


@pytest.mark.parametrize("dtype", CACHES)
def test_long_sequences_shared_by_many_warps(dtype):
    import qwantize_b200 as q
    c, codes, table, lengths = setup(3, [70000, 33, 9000], 1, 128, dtype, 5)
    x = queries(3, 4, 128, torch.bfloat16, 6)
    out = q.kv_cache_attention(c, x, table, lengths)
    check(out, x, *codes, table, lengths)
    assert all(torch.equal(out, q.kv_cache_attention(c, x, table, lengths)) for _ in range(3))


@pytest.mark.parametrize("dtype", CACHES)
def test_what_lies_behind_the_last_token_does_not_count(dtype):
    """Codes behind a sequence's end, infinities and NaN of E4M3 among them, and
    scales of pages that no token is in."""
    import qwantize_b200 as q
    c, (k, ks, v, vs), table, lengths = setup(2, [70, 130], 2, 64, dtype, 7, extra=2)
    x = queries(2, 4, 64, torch.float16, 8)
    out = q.kv_cache_attention(c, x, table, lengths)
    k, v, ks, vs = k.clone(), v.clone(), ks.clone(), vs.clone()
    for b, n in enumerate((70, 130)):
        last = int(table[b, n // 64])
        for codes in (k, v):
            codes.view(torch.uint8)[last, :, n % 64:] = 0x7F
            for later in table[b, n // 64 + 1:].tolist():
                codes.view(torch.uint8)[later] = 0xFF
        for later in table[b, n // 64 + 1:].tolist():
            ks[later] = vs[later] = float("nan")
    c.load_codes(k, ks, v, vs)
    assert torch.equal(q.kv_cache_attention(c, x, table, lengths), out)


def test_scale_large_scores_and_shared_pages():
    import qwantize_b200 as q
    c, codes, table, lengths = setup(2, [200, 256], 2, 128, torch.int8, 9)
    table[1, :2] = table[0, :2]  # a shared prefix
    x = queries(2, 8, 128, torch.bfloat16, 10)
    for scale in (0.0, -0.05, 1.0, 30.0):
        check(q.kv_cache_attention(c, x, table, lengths, scale=scale), x, *codes, table, lengths, scale)
    for mag in (2.0**-90, 2.0**60):
        check(q.kv_cache_attention(c, x * mag, table, lengths, scale=1.0 / mag), x * mag, *codes, table, lengths, 1.0 / mag)


def test_pages_that_the_cache_does_not_have_are_skipped():
    import qwantize_b200 as q
    c, (k, ks, v, vs), table, lengths = setup(2, [150, 100], 2, 128, torch.int8, 11)
    x = queries(2, 4, 128, torch.bfloat16, 12)
    table[0, 1] = -1
    table[1, :] = c.num_pages
    out = q.kv_cache_attention(c, x, table, lengths)
    assert not out[1].any()
    # sequence 0 without its second page
    t2 = torch.stack((table[0, 0], table[0, 2]))[None].contiguous()
    n2 = torch.tensor([64 + 150 - 128], dtype=torch.int32, device=DEV)
    check(out[:1], x[:1], k, ks, v, vs, t2, n2)
    long = torch.tensor([10**6, -5], dtype=torch.int32, device=DEV)  # beyond the table: what it has; negative: none
    table[0, 1] = table[0, 0]
    out = q.kv_cache_attention(c, x, table, long)
    check(out[:1], x[:1], k, ks, v, vs, table[:1], long[:1])
    assert not out[1].any()


def test_strides_streams_and_int64_indices():
    import qwantize_b200 as q
    c, codes, table, lengths = setup(4, [70, 1, 200, 64], 2, 64, torch.int8, 13)
    qkv = queries(4, 12, 64, torch.bfloat16, 14)
    x = qkv[:, 2:10].contiguous()
    base = q.kv_cache_attention(c, x, table, lengths)
    assert torch.equal(q.kv_cache_attention(c, qkv[:, 2:10], table, lengths), base)
    assert torch.equal(q.kv_cache_attention(c, x.transpose(0, 1).contiguous().transpose(0, 1), table, lengths), base)
    assert torch.equal(q.kv_cache_attention(c, x, table.long(), lengths.long()), base)
    wide = torch.zeros(4, table.shape[1] + 5, dtype=torch.int32, device=DEV)
    wide[:, : table.shape[1]] = table
    assert torch.equal(q.kv_cache_attention(c, x, wide[:, : table.shape[1]], lengths), base)
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].reshape(x.shape)
    odd.copy_(x)
    assert torch.equal(q.kv_cache_attention(c, odd, table, lengths), base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [q.kv_cache_attention(c, x, table, lengths) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(v, base) for v in again)
    assert q.kv_cache_attention(c, x[:0], table[:0], lengths[:0]).shape == (0, 8, 64)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes: the last pages hold the tokens."""
    import qwantize_b200 as q
    P, H, D = 270000, 2, 128  # 4.4e9 bytes of keys
    c = q.KVCache8(P, H, D)
    small, k, ks, v, vs = fill(4, H, D, torch.int8, 15)
    c.k[-4:], c.v[-4:], c.k_scale[-4:], c.v_scale[-4:] = small.k, small.v, small.k_scale, small.v_scale
    table = torch.tensor([[3, 0, 2]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([150], dtype=torch.int32, device=DEV)
    x = queries(1, 4, D, torch.bfloat16, 16)
    assert torch.equal(q.kv_cache_attention(c, x, table + (P - 4), lengths), q.kv_cache_attention(small, x, table, lengths))
    new = queries(1, H, D, torch.bfloat16, 17)
    for cache, t in ((c, table + (P - 4)), (small, table)):
        q.kv_cache_append(cache, new, new, t, lengths)
    for a, b in zip(q.kv_cache_read(c, table[0] + (P - 4)), q.kv_cache_read(small, table[0])):
        assert torch.equal(a, b)
    del c


# --- append and read -------------------------------------------------------------


def appended(codes, scale, new, table, old, counts, dtype):
    """The oracle: codes (P, H, 64, D) and scales after the append, fp32 steps."""
    codes, scale = codes.clone(), scale.clone()
    at = 0
    for b, (o, n) in enumerate(zip(old, counts)):
        x = new[at: at + n].float()
        at += n
        for blk in range(o // 64, -(-(o + n) // 64) if n else o // 64):
            lo, hi = max(o, 64 * blk), min(o + n, 64 * blk + 64)
            page, off = int(table[b, blk]), lo - 64 * blk
            y = x[lo - o: hi - o].transpose(0, 1)  # (H, tokens, D)
            before = scale[page] if off else torch.zeros_like(scale[page])
            s = torch.maximum(before, y.abs().amax((1, 2)) * torch.tensor(1 / TOP[dtype]))  # the factor rounded to fp32
            ratio = torch.where(s > 0, before / s, torch.zeros_like(s))
            block = torch.zeros(codes.shape[1:], dtype=torch.float32)
            block[:, :off] = encode(codes[page, :, :off].float() * ratio[:, None, None], dtype).float()
            q = torch.where(s[:, None, None] > 0, y / s[:, None, None], torch.zeros_like(y))
            block[:, off: hi - 64 * blk] = encode(q, dtype).float()
            codes[page] = block.to(dtype)
            scale[page] = s
    return codes, scale


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("old,counts,H", [
    ([0], [1], 1), ([5], [1], 2), ([63], [1], 3), ([64], [1], 1), ([0], [64], 2), ([0], [65], 1), ([1], [63], 2), ([63], [130], 2),
    ([10, 0, 64, 100], [1, 1, 1, 1], 8), ([10, 0, 7, 128, 50], [200, 0, 3, 64, 1], 4)])
def test_append_and_read(dtype, D, old, counts, H):
    import qwantize_b200 as q
    B = len(old)
    ends = [o + n for o, n in zip(old, counts)]
    c, (k, ks, v, vs), table, lengths = setup(B, ends, H, D, dtype, sum(old) + H)
    lengths = torch.tensor(old, dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(20)
    for t, mag in ((torch.bfloat16, 1.0), (torch.float16, 0.01), (torch.bfloat16, 100.0)):
        nk, nv = ((mag * torch.randn(sum(counts), H, D, generator=g)).to(t) for _ in range(2))
        if counts == [1] * B:
            q.kv_cache_append(c, nk.to(DEV), nv.to(DEV), table, lengths)
        else:
            cu = torch.tensor([0] + counts).cumsum(0).int().to(DEV)
            q.kv_cache_append(c, nk.to(DEV), nv.to(DEV), table, lengths, cu_new=cu, max_new=max(counts))
        k, ks = appended(k, ks, nk, table.cpu(), old, counts, dtype)
        v, vs = appended(v, vs, nv, table.cpu(), old, counts, dtype)
        ck, cks, cv, cvs = (x.cpu() for x in c.codes())
        assert torch.equal(cks, ks) and torch.equal(cvs, vs)
        assert torch.equal(ck.float(), k.float()) and torch.equal(cv.float(), v.float())
    pages = torch.randperm(c.num_pages, generator=g).int().to(DEV)
    rk, rv = q.kv_cache_read(c, pages)
    p = pages.cpu().long()
    assert torch.equal(rk.cpu(), k[p].float() * ks[p][..., None, None])
    assert torch.equal(rv.cpu(), v[p].float() * vs[p][..., None, None])
    for t in (torch.bfloat16, torch.float16):
        a, b = q.kv_cache_read(c, pages, t)
        assert torch.equal(a, rk.to(t)) and torch.equal(b, rv.to(t))


def test_append_then_attend_token_by_token():
    """130 tokens one at a time from an empty cache: at every step the codes and
    scales of the oracle, then attention over them."""
    import qwantize_b200 as q
    B, H, D, n = 2, 2, 64, 130
    g = torch.Generator().manual_seed(21)
    k, v = (torch.randn(n, B, H, D, generator=g).to(torch.bfloat16) for _ in range(2))
    x = torch.randn(B, 4, D, generator=g).to(torch.bfloat16).to(DEV)
    for dtype in CACHES:
        c = q.KVCache8(8, H, D, dtype)
        table = torch.tensor([[5, 0, 3], [1, 7, 2]], dtype=torch.int32, device=DEV)
        lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
        rk, rks, rv, rvs = (t.cpu() for t in c.codes())
        for i in range(n):
            q.kv_cache_append(c, k[i].to(DEV), v[i].to(DEV), table, lengths)
            rk, rks = appended(rk, rks, k[i], table.cpu(), [i] * B, [1] * B, dtype)
            rv, rvs = appended(rv, rvs, v[i], table.cpu(), [i] * B, [1] * B, dtype)
            lengths += 1
            if i % 13 == 0 or i == n - 1:
                ck, cks, cv, cvs = (t.cpu() for t in c.codes())
                assert torch.equal(cks, rks) and torch.equal(cvs, rvs)
                assert torch.equal(ck.float(), rk.float()) and torch.equal(cv.float(), rv.float())
        check(q.kv_cache_attention(c, x, table, lengths), x, rk, rks, rv, rvs, table, lengths)


def test_append_zeros_and_non_finite_values():
    import qwantize_b200 as q
    c = q.KVCache8(4, 2, 64)
    table = torch.tensor([[2], [0]], dtype=torch.int32, device=DEV)
    lengths = torch.zeros(2, dtype=torch.int32, device=DEV)
    z = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    q.kv_cache_append(c, z, z, table, lengths)
    assert not c.k_scale.any() and not c.k.any()
    out = q.kv_cache_attention(c, z + 1, table, lengths + 1)
    assert not out.any()
    bad = z + 1
    bad[0, 1, 5] = float("inf")
    q.kv_cache_append(c, bad, z, table, lengths + 1)
    k, v = q.kv_cache_read(c, torch.tensor([2, 0, 9], dtype=torch.int32, device=DEV))
    assert bool(k[0, 1].isnan().all()) and bool(torch.isfinite(k[0, 0]).all()) and bool(torch.isfinite(k[1]).all())
    assert bool(k[2].isnan().all()) and not v[:2].any()
    q.kv_cache_append(c, z + 1, z, table, lengths + 2)  # a page stays marked
    assert bool(c.k_scale[2, 1].isnan()) and not c.k[2, 1].any()
    q.kv_cache_append(c, z + 1, z, table, lengths)      # until it is begun again
    assert bool(torch.isfinite(c.k_scale).all())


def test_append_strides_bounds_and_limits():
    import qwantize_b200 as q
    g = torch.Generator().manual_seed(22)
    kv = torch.randn(6, 12, 64, generator=g).to(torch.float16).to(DEV)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([62, 0], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 5, 6], dtype=torch.int32, device=DEV)
    a, b = q.KVCache8(4, 4, 64), q.KVCache8(4, 4, 64)
    q.kv_cache_append(a, kv[:, :4], kv[:, 4:8], table, lengths, cu_new=cu)
    q.kv_cache_append(b, kv[:, :4].contiguous(), kv[:, 4:8].contiguous(), table.long(), lengths, cu_new=cu.long(), max_new=5)
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.k_scale, b.k_scale)
    before = a.k.clone()
    # positions beyond the table and pages that do not exist are not written
    q.kv_cache_append(a, kv[:2, :4], kv[:2, :4], table, torch.tensor([128, 500], dtype=torch.int32, device=DEV))
    q.kv_cache_append(a, kv[:2, :4], kv[:2, :4], table - 100, lengths)
    assert torch.equal(a.k, before)


def test_refusals():
    import qwantize_b200 as q
    c = q.KVCache8(4, 2, 64)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    n = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    for kwargs in (dict(head_dim=96), dict(dtype=torch.uint8), dict(kv_heads=0)):
        with pytest.raises(AssertionError):
            q.KVCache8(**{**dict(num_pages=4, kv_heads=2, head_dim=64), **kwargs})
    for args in ((c, x[:, :1], x, table, n), (c, x.float(), x.float(), table, n), (c, x, x, table, n[:0]),
                 (c, x, x, table.float(), n), (c, torch.cat((x, x)), torch.cat((x, x)), table, n), (x, x, x, table, n)):
        with pytest.raises(AssertionError):
            q.kv_cache_append(*args)
    for args in ((c, x[:, :, :32], table, n), (c, torch.cat((x, x[:, :1]), 1), table, n), (c, x.float(), table, n),
                 (c, x, table, n.cpu())):
        with pytest.raises(AssertionError):
            q.kv_cache_attention(*args)
    with pytest.raises(AssertionError):
        q.kv_cache_read(c, n, torch.float64)
    with pytest.raises(AssertionError):
        c.load_codes(c.codes()[0][:2], c.k_scale, c.codes()[2], c.v_scale)
