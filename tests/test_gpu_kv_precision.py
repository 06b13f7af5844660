"""What attention over the 8-bit cache keeps of small probabilities.

The bounds are those of the other attention tests but for the probabilities: they
are rounded to fp16 at 2^14 or more times their value over the largest, so one is
off by 2^-11 of itself, or by half a subnormal step, at most 2^-25 / 2^14 = 2^-39 of
the largest."""
import pytest
import torch

from tests.test_gpu_kv_cache import CACHES, U, encode
from tests.test_gpu_linear import ROUND

pytestmark = pytest.mark.gpu
DEV = "cuda"


def limits(q, k, ks, v, vs, table, n, p_round):
    """Output and error bound in 64 bits; one sequence, one cache head."""
    D = q.shape[2]
    pages = table[0, : -(-n // 64)].long().cpu()
    kk, vv = ((c[pages].double() * s[pages].double()[..., None, None]).transpose(0, 1).reshape(-1, D)[:n] for c, s in ((k, ks), (v, vs)))
    qq = q[0].cpu().double()
    scale = D**-0.5
    s = qq @ kk.T * scale
    es = scale * D * 2 * U * (qq.abs() @ kk.abs().T) + 4 * U * s.abs() + 4 * U * (s - s.amax(-1, keepdim=True)).abs()
    p = torch.softmax(s, -1)
    rel = torch.expm1(2 * es.amax(-1, keepdim=True)) + p_round + 2 * U * n + 8 * U
    ref = p @ vv
    lim = rel * (p @ vv.abs()) + 2.0**-39 * p.amax(-1, keepdim=True) * vv.abs().sum(0)
    return ref, lim


def check(out, ref, lim):
    lim = lim + ROUND[out.dtype] * (ref.abs() + lim) + (2.0**-25 if out.dtype == torch.float16 else 1e-30)
    err = (out[0].cpu().double() - ref).abs()
    assert bool((err <= lim).all()), (float((err / lim).max()), int((err > lim).sum()))


def cached(D, n, dtype, seed, extra=0):
    """Pages in a random order for n tokens, and what names them."""
    import qwantize_b200 as q
    P = -(-n // 64)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(P, generator=g).int().reshape(1, P)
    wide = torch.cat([table, table.new_full((1, extra), -1)], 1).to(DEV)
    return q.KVCache8(P, 1, D, dtype), table, wide, torch.tensor([n], dtype=torch.int32, device=DEV), g


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,extra", [(2000, 0), (2000, 130), (30000, 0)])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("gap", [14.0, 16.5, 17.5, 20.0])
def test_one_dominant_token_and_many_small_ones(dtype, D, n, extra, last, gap):
    """A token that takes nearly all of the weight and has the value zero: the output
    is the sum of thousands of probabilities below 2^-20 of the largest."""
    import qwantize_b200 as q
    if D == 128 and n == 2000 and not extra:
        n = 1500  # at most two pages for each warp of a pair's CTA
    c, table, wide, lengths, g = cached(D, n, dtype, n + int(gap), extra)
    P = c.num_pages
    at = n - 1 if last else 3
    page, slot = int(table[0, at // 64]), at % 64
    k = encode(torch.randn(P, 1, 64, D, generator=g), dtype)
    ks = torch.full((P, 1), 1.0 / 64)
    top = 96.0
    k[page, 0] = 0
    k[page, 0, slot] = encode(torch.full((D,), top), dtype)
    ks[page, 0] = gap / (D**0.5 * top)
    v = encode(60 + 30 * torch.randn(P, 1, 64, D, generator=g), dtype)
    v[page, 0, slot] = 0
    vs = torch.full((P, 1), 40.0)
    c.load_codes(k, ks, v, vs)
    for t in (torch.bfloat16, torch.float16):
        x = torch.ones(1, 3, D, dtype=t, device=DEV)
        x[0, 1] *= 0.97
        out = q.kv_cache_attention(c, x, wide, lengths)
        check(out, *limits(x, k, ks, v, vs, table, n, 2.0**-11))


@pytest.mark.parametrize("dtype", CACHES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,extra", [(2, 0), (70, 0), (2, 200), (2000, 200)])
@pytest.mark.parametrize("heads", [5, 16])
def test_fp16_results_of_values_that_nearly_cancel(dtype, D, n, extra, heads):
    """fp16 results keep 11 bits, as many as a probability rounded to fp16: there the
    remainder counts too, which leaves 2^-22 of it.  Two tokens of nearly the same
    weight and opposite values show it."""
    import qwantize_b200 as q
    c, table, wide, lengths, g = cached(D, n, dtype, n + heads, extra)
    P = c.num_pages
    k = torch.zeros(P, 1, 64, D)
    ks = torch.full((P, 1), 0.02 / (8 * D**0.5))  # a score is 0.0025 a code
    v, vs = torch.zeros(P, 1, 64, D), torch.full((P, 1), 0.25)
    value = torch.tensor([64.0, -80, 96, 112])[torch.randint(4, (D,), generator=g)]
    for i, code, sign in ((0, 96.0, 1), (n - 1, 88.0, -1)):
        page, slot = int(table[0, i // 64]), i % 64
        k[page, 0, slot], v[page, 0, slot] = code, sign * value
    k, v = encode(k, dtype), encode(v, dtype)
    c.load_codes(k, ks, v, vs)
    x = (torch.linspace(0.5, 2.5, heads)[:, None] * torch.ones(D)).to(torch.float16)[None].to(DEV)
    check(q.kv_cache_attention(c, x, wide, lengths), *limits(x, k, ks, v, vs, table, n, 2.0**-22))
