"""fp4_moe against the definition in 64 bits.

The oracle decodes the packed experts and runs the layer in double on the CPU.
Tolerances, with u = 2^-24 (fp32) and h = 2^-11 (fp16 significand):
* logits: H u sum |x r|; weights follow by the softmax's derivative (at most the
  logit error times 2) plus a few u;
* gate and up: H 2u sum |w x|; the activation is a product of them, its
  derivative at most 1.1 |up| and |gate|; it is rounded to fp16 relative to the row's
  largest (h |a| plus 2^-25 2^-14 of it, nothing beside h);
* down: I 2u sum |w a| plus the activation's error through |w|; then the weights'
  error, and one rounding of the result (2^-8 bf16, 2^-11 fp16)."""
import pytest
import torch

from tests.test_gpu_linear import BLOCK, ROUND, decode

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0**-24


def make(E, H, I, fmt, seed):
    import qwantize_b200 as q
    g = torch.Generator().manual_seed(seed)
    up = torch.randn(E, 2 * I, H, generator=g) * torch.exp(0.5 * torch.randn(E, 2 * I, 1, generator=g)) / H**0.5
    down = torch.randn(E, H, I, generator=g) / I**0.5
    fn = q.nvfp4_quantize_packed if fmt == "nvfp4" else q.mxfp4_quantize_packed
    bs, t = BLOCK[fmt], 2.0**-6 if fmt == "nvfp4" else 1.0
    pack = lambda w: fn((w / t).to(DEV, torch.bfloat16).reshape(*w.shape[:-1], -1, bs))  # noqa: E731
    return pack(up), pack(down), t


def oracle(x, router, up, down, fmt, t, top, renorm, ids):
    """Output, weights and their error bounds, with the kernel's own choice of
    experts (checked apart)."""
    x, r = x.cpu().double(), router.cpu().double()
    H = x.shape[1]
    logits = x @ r.T
    el = H * U * (x.abs() @ r.abs().T)
    ids = ids.cpu().long()
    chosen = logits.gather(1, ids)
    base = chosen if renorm else logits
    w = torch.exp(chosen - torch.logsumexp(base, -1, keepdim=True))
    ew = w * (2 * el.amax(-1, keepdim=True) + 40 * U) + 1e-30
    y, ey = torch.zeros_like(x), torch.zeros_like(x)
    for e in ids.unique().tolist():
        rows, nth = torch.nonzero(ids == e, as_tuple=True)
        wu, wd = decode(up[0][e], up[1][e], fmt, t), decode(down[0][e], down[1][e], fmt, t)
        I = wd.shape[1]
        h, eh = x[rows] @ wu.T, 2 * U * H * (x[rows].abs() @ wu.abs().T)
        gate, upv = h[:, :I], h[:, I:]
        a = gate * torch.sigmoid(gate) * upv
        ea = 1.1 * eh[:, :I] * upv.abs() + (gate.abs() + 0.3) * eh[:, I:] + (2.0**-11 + 8 * U) * a.abs() + 2.0**-38 * a.abs().amax(-1, keepdim=True)
        d = a @ wd.T
        ed = ea @ wd.abs().T + 2 * U * I * (a.abs() @ wd.abs().T)
        c, ec = w[rows, nth, None], ew[rows, nth, None]
        y[rows] += c * d
        ey[rows] += c * ed + ec * d.abs() + 4 * U * c * d.abs()
    return y, ey, w, ew, logits, el


def check(x, router, up, down, fmt, t, top, renorm=True):
    import qwantize_b200 as q
    ex = q.FP4Experts(up, down, fmt, tensor_scales=(t, t))
    out, ids, w = q.fp4_moe(x, router, ex, top, renormalize=renorm, return_routing=True)
    y, ey, rw, ew, logits, el = oracle(x, router, up, down, fmt, t, top, renorm, ids)
    # the experts taken are the largest logits, in descending order, within the logits' error
    got = logits.gather(1, ids.cpu().long())
    best = logits.topk(top, dim=-1).values
    tol = 2 * el.amax(-1, keepdim=True) + 1e-30
    assert bool(((got - best).abs() <= tol).all())
    assert all(len(set(r)) == top for r in ids.cpu().tolist())
    assert bool(((w.cpu().double() - rw).abs() <= ew).all())
    err = (out.cpu().double() - y).abs()
    lim = ey + ROUND[out.dtype] * (y.abs() + ey) + (2.0**-25 if out.dtype == torch.float16 else 1e-30)
    assert bool((err <= lim).all()), (float((err / lim).max()), int((err > lim).sum()))
    return ex, out, ids, w


def tokens(T, H, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, H, generator=g) * torch.exp(0.5 * torch.randn(H, generator=g))).to(dtype).to(DEV)


def router_of(E, H, dtype, seed):
    return (torch.randn(E, H, generator=torch.Generator().manual_seed(seed)) / H**0.5).to(dtype).to(DEV)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("T,H,I,E,top", [
    (1, 32, 32, 1, 1), (1, 256, 96, 8, 2), (1, 2048, 768, 16, 8), (2, 96, 160, 3, 3), (7, 544, 224, 13, 4),
    (8, 128, 64, 4, 1), (9, 320, 96, 2, 2), (17, 256, 416, 8, 2), (33, 160, 96, 5, 2), (64, 512, 128, 64, 8),
    (64, 96, 96, 2, 1), (64, 64, 32, 1, 1), (5, 64, 32, 200, 16), (3, 64, 32, 512, 5)])
def test_moe_shapes(fmt, T, H, I, E, top):
    up, down, t = make(E, H, I, fmt, T + H + I + E)
    for k, (dtype, rdtype) in enumerate([(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.bfloat16, torch.float16)]):
        check(tokens(T, H, dtype, k), router_of(E, H, rdtype, k), up, down, fmt, t, top)


@pytest.mark.parametrize("renorm", [True, False])
def test_softmax_over_all_or_over_the_chosen(renorm):
    up, down, t = make(12, 128, 64, "nvfp4", 3)
    check(tokens(20, 128, torch.bfloat16, 1), router_of(12, 128, torch.float32, 2), up, down, "nvfp4", t, 3, renorm)


def test_ties_take_the_lowest_index():
    import qwantize_b200 as q
    up, down, t = make(40, 64, 32, "nvfp4", 4)
    ex = q.FP4Experts(up, down, tensor_scales=(t, t))
    x = tokens(6, 64, torch.bfloat16, 5)
    zero = torch.zeros(40, 64, dtype=torch.bfloat16, device=DEV)
    _, ids, w = q.fp4_moe(x, zero, ex, 4, return_routing=True)
    assert ids.tolist() == [[0, 1, 2, 3]] * 6 and bool((w == 0.25).all())
    r = router_of(40, 64, torch.bfloat16, 6)
    r[7] = r[33] = r[2]
    logits = x.double() @ r.double().T
    _, ids, _ = q.fp4_moe(x, r, ex, 16, return_routing=True)
    for row, lg in zip(ids.tolist(), logits.tolist()):
        same = [e for e in row if e in (2, 7, 33)]
        assert same == sorted(same)


def test_many_tokens_on_one_expert():
    """All 64 tokens on one expert: its weights are read for two groups of 32."""
    up, down, t = make(6, 96, 64, "nvfp4", 7)
    x = tokens(64, 96, torch.bfloat16, 8).abs()
    r = -router_of(6, 96, torch.float32, 9).abs()
    r[4] = -r[4]
    _, _, ids, _ = check(x, r, up, down, "nvfp4", t, 1)
    assert ids.unique().tolist() == [4]


@pytest.mark.parametrize("scale", [2.0**-70, 2.0**-20, 2.0**40])
def test_bf16_tokens_of_any_magnitude(scale):
    """bf16 reaches beyond fp16: tokens and activations carry a power of two."""
    import qwantize_b200 as q
    up, down, t = make(4, 64, 96, "mxfp4", 10)
    ex = q.FP4Experts(up, down, "mxfp4")
    x = tokens(3, 64, torch.bfloat16, 11) * scale
    zero = torch.zeros(4, 64, device=DEV)
    out, ids, w = q.fp4_moe(x, zero, ex, 2, return_routing=True)
    y, ey, *_ = oracle(x, zero, up, down, "mxfp4", 1.0, 2, True, ids)
    err = (out.cpu().double() - y).abs()
    assert bool((err <= ey + 2.0**-8 * (y.abs() + ey) + 2.0**-133).all())


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_a_token_with_a_non_finite_value_spoils_no_other(bad):
    import qwantize_b200 as q
    up, down, t = make(8, 128, 64, "nvfp4", 12)
    ex = q.FP4Experts(up, down, tensor_scales=(t, t))
    r = router_of(8, 128, torch.bfloat16, 13)
    x = tokens(10, 128, torch.bfloat16, 14)
    good = q.fp4_moe(x, r, ex, 2)
    x[3, 77] = bad
    y, ids, _ = q.fp4_moe(x, r, ex, 2, return_routing=True)
    rest = [i for i in range(10) if i != 3]
    assert torch.equal(y[rest], good[rest]) and not bool(torch.isfinite(y[3]).all())
    assert bool(((ids >= 0) & (ids < 8)).all())


def test_strides_shapes_streams_and_repeats():
    import qwantize_b200 as q
    up, down, t = make(8, 128, 64, "nvfp4", 15)
    ex = q.FP4Experts(up, down, tensor_scales=(t, t))
    r = router_of(8, 128, torch.bfloat16, 16)
    wide = tokens(24, 264, torch.bfloat16, 17)
    x = wide[:, 64:192].contiguous()
    base = q.fp4_moe(x, r, ex, 3)
    assert torch.equal(q.fp4_moe(wide[:, 64:192], r, ex, 3), base)
    assert torch.equal(q.fp4_moe(x.T.contiguous().T, r, ex, 3), base)
    assert torch.equal(q.fp4_moe(x.reshape(2, 12, 128), r, ex, 3).reshape(24, 128), base)
    assert torch.equal(q.fp4_moe(x.cpu(), r, ex, 3), base.cpu())
    assert torch.equal(q.fp4_moe(x[5], r, ex, 3), q.fp4_moe(x[5:6], r, ex, 3)[0])
    out = torch.empty_like(x)
    assert q.fp4_moe(x, r, ex, 3, out=out).data_ptr() == out.data_ptr() and torch.equal(out, base)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [q.fp4_moe(x, r, ex, 3) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(v, base) for v in again)
    assert q.fp4_moe(x[:0], r, ex, 3).shape == (0, 128)


def test_quantize_experts():
    import qwantize_b200 as q
    g = torch.Generator().manual_seed(18)
    up, down = torch.randn(4, 128, 64, generator=g) * 0.05, torch.randn(4, 64, 64, generator=g) * 0.05
    x, r = tokens(5, 64, torch.bfloat16, 19), router_of(4, 64, torch.bfloat16, 20)
    for fmt in ("nvfp4", "mxfp4"):
        for method in ("naive", "optimal"):
            out, ids, w = q.fp4_moe(x, r, q.FP4Experts.quantize(up.to(DEV, torch.bfloat16), down.to(DEV, torch.bfloat16), fmt, method), 2,
                                    return_routing=True)
            ref = torch.zeros(5, 64, dtype=torch.float64)
            for t in range(5):
                for e, c in zip(ids[t].tolist(), w[t].tolist()):
                    h = x[t].cpu().double() @ up[e].double().T
                    ref[t] += c * ((torch.nn.functional.silu(h[:64]) * h[64:]) @ down[e].double().T)
            # three products with weights that FP4 moves by about 0.1 each
            assert float((out.cpu().double() - ref).norm() / ref.norm()) < 0.4


def test_refusals():
    import qwantize_b200 as q
    up, down, t = make(4, 64, 32, "nvfp4", 21)
    ex = q.FP4Experts(up, down)
    r = router_of(4, 64, torch.bfloat16, 22)
    x = tokens(2, 64, torch.bfloat16, 23)
    for args in ((x[:, :32], r, ex, 1), (x.float(), r, ex, 1), (x, r[:3], ex, 1), (x, r, ex, 5), (x, r, ex, 0), (x, r, up, 1),
                 (tokens(65, 64, torch.bfloat16, 1), r, ex, 1), (x, r.double(), ex, 1)):
        with pytest.raises(AssertionError):
            q.fp4_moe(*args)
    with pytest.raises(AssertionError):
        q.FP4Experts(up, up)
    with pytest.raises(AssertionError):
        q.FP4Experts((up[0][0], up[1][0]), (down[0][0], down[1][0]))
    with pytest.raises(AssertionError):
        q.FP4Experts.quantize(torch.zeros(2, 48, 32, device=DEV), torch.zeros(2, 32, 24, device=DEV))
