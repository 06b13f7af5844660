"""fp4_linear against the definition in 64 bits.

The oracle decodes the packed weight and quantizes the activations in double
precision on the CPU, then multiplies.  Each product of two E2M1 codes and two
scales is exact in fp32, and the kernel sums K of them (and the splits of K) in
fp32 in some order, possibly truncating: an element is within
K * 2^-23 * sum |terms| of the exact sum.  A 16-bit result adds one rounding:
half a step of its significand, 2^-8 (bf16: 8 bits) or 2^-11 (fp16: 11 bits) of its magnitude, or half an fp16 subnormal step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def decode(codes, packed, fmt, t=1.0):
    c = codes.cpu()
    s = c.view(torch.float8_e4m3fn).double() if fmt == "nvfp4" else torch.exp2(c.double() - 127)
    p = packed.cpu().reshape(*c.shape[:-1], -1).long()
    v = torch.stack((VALUES[p & 15], VALUES[p >> 4]), -1).flatten(-2)
    return (v.reshape(*c.shape, -1) * s[..., None]).flatten(-2) * t


def quantized_rows(x, fmt):
    """The naive FP4 form of each row, in double."""
    x = x.cpu().double()
    amax = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax / 2688)
    t = torch.where(amax > 0, torch.exp2(torch.where(m == 0.5, e - 1, e).clamp(min=-120).double()), torch.ones_like(amax))
    if fmt == "mxfp4":
        t = torch.ones_like(t)
    b = (x / t).reshape(x.shape[0], -1, BLOCK[fmt])
    amax = b.abs().amax(-1, keepdim=True)
    if fmt == "nvfp4":
        s = (amax.float() / 6).to(torch.float8_e4m3fn).double()
    else:
        s = torch.exp2(torch.frexp(amax.clamp(min=1e-30))[1].double() - 3)
    a = b.abs() / torch.where(s > 0, s, torch.ones_like(s)) * (s > 0)
    q = VALUES[torch.bucketize(a, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64))]
    return (torch.sign(b) * q * s).reshape(x.shape) * t


def make_weight(N, K, fmt, seed):
    import qwantize_b200 as q
    g = torch.Generator().manual_seed(seed)
    W = torch.randn(N, K, generator=g) * torch.exp(torch.randn(N, 1, generator=g))
    fn = q.nvfp4_quantize_packed if fmt == "nvfp4" else q.mxfp4_quantize_packed
    return fn(W.to(DEV, torch.bfloat16).reshape(N, K // BLOCK[fmt], BLOCK[fmt]))


def acts(T, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, K, generator=g) * torch.exp(torch.randn(K, generator=g)) * torch.exp(torch.randn(T, 1, generator=g))).to(dtype)


def check(y, x, codes, packed, fmt, t=1.0, bias=None):
    xq, w = quantized_rows(x, fmt), decode(codes, packed, fmt, t)
    ref = xq @ w.T
    tol = x.shape[-1] * 2.0**-23 * (xq.abs() @ w.abs().T)
    if bias is not None:
        ref = ref + bias.cpu().double()
        tol = tol + 2.0**-23 * ref.abs()
    tol = tol + ROUND[y.dtype] * (ref.abs() + tol) + (2.0**-25 if y.dtype == torch.float16 else 0.0)
    over = ref.to(y.dtype).isinf()  # beyond the type's range the rounded result is infinite
    assert torch.equal(y.cpu()[over], ref.to(y.dtype)[over])
    err = torch.where(over, torch.zeros_like(ref), (y.cpu().double() - ref).abs())
    assert bool((err <= tol + 1e-30).all()), (float((err / (tol + 1e-30)).max()), int((err > tol + 1e-30).sum()))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("T,K,N", [
    (1, 32, 1), (1, 256, 128), (1, 2560, 300), (2, 288, 7), (5, 2560, 1000), (16, 1024, 129), (17, 96, 640),
    (33, 512, 256), (64, 2560, 128), (65, 800, 333), (128, 1056, 520), (130, 256, 257), (300, 2560, 1000),
    (513, 96, 768), (1025, 544, 31)])
def test_linear_shapes(fmt, T, K, N):
    import qwantize_b200 as q
    codes, packed = make_weight(N, K, fmt, T + K + N)
    w = q.FP4Weight(codes, packed, fmt)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = acts(T, K, dtype, T).to(DEV)
        check(q.fp4_linear(x, w), x, codes, packed, fmt)
    check(q.fp4_linear(x, w, out_dtype=torch.bfloat16), x, codes, packed, fmt)


@pytest.mark.parametrize("T", [1, 3, 40, 200])
@pytest.mark.parametrize("K", [16, 48, 240, 272, 2544])
def test_nvfp4_odd_block_counts(T, K):
    """K a multiple of 16 but not of 32: packed rows are padded to 16 bytes."""
    import qwantize_b200 as q
    codes, packed = make_weight(77, K, "nvfp4", K)
    w = q.FP4Weight(codes, packed, tensor_scale=0.125)
    x = acts(T, K, torch.bfloat16, K).to(DEV)
    check(q.fp4_linear(x, w, out_dtype=torch.float32), x, codes, packed, "nvfp4", 0.125)


@pytest.mark.parametrize("fmt,K", [("nvfp4", 16), ("nvfp4", 272), ("nvfp4", 9744), ("mxfp4", 32), ("mxfp4", 2592), ("mxfp4", 9728), ("nvfp4", 40960)])
@pytest.mark.parametrize("N", [77, 1500])
def test_a_single_token_like_a_row_of_two(fmt, K, N):
    """One token is quantized by the product's own kernel: the same bits as from
    the row in a batch, whatever the type, the magnitude and what is not finite."""
    import qwantize_b200 as q
    codes, packed = make_weight(N, K, fmt, K + N)
    w = q.FP4Weight(codes, packed, fmt)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x = acts(2, K, dtype, K).to(DEV)
        check(q.fp4_linear(x[:1], w), x[:1], codes, packed, fmt)
        rows = [x[0], x[0] * 0, x[0] * 2.0**-10, x[0] * 2.0**5]
        if dtype != torch.float16:
            rows += [x[0] * 2.0**70, x[0] * 2.0**-70]
        for bad in (float("inf"), float("nan")):
            rows.append(x[0].clone())
            rows[-1][K // 2] = bad
        for r in rows:
            pair = torch.stack([r, x[1]])
            one, two = q.fp4_linear(pair[:1], w), q.fp4_linear(pair, w)[:1]
            assert torch.equal(one.isnan(), two.isnan()) and torch.equal(one.nan_to_num(), two.nan_to_num())


def test_many_tiles_and_bands():
    """More tiles than SMs, several bands of token tiles, a ragged last one."""
    import qwantize_b200 as q
    codes, packed = make_weight(2700, 288, "nvfp4", 1)
    w = q.FP4Weight(codes, packed)
    x = acts(4500, 288, torch.float16, 2).to(DEV)
    check(q.fp4_linear(x, w, out_dtype=torch.float32), x, codes, packed, "nvfp4")


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("bias_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T", [1, 37, 400])
def test_bias_out_and_leading_dimensions(fmt, bias_dtype, T):
    import qwantize_b200 as q
    codes, packed = make_weight(96, 320, fmt, 3)
    w = q.FP4Weight(codes, packed, fmt)
    bias = torch.randn(96, generator=torch.Generator().manual_seed(9)).to(bias_dtype).to(DEV)
    x = acts(2 * T, 320, torch.bfloat16, 4).to(DEV).reshape(2, T, 320)
    out = torch.full((2, T, 96), float("nan"), dtype=torch.float32, device=DEV)
    y = q.fp4_linear(x, w, bias=bias, out=out)
    assert y.data_ptr() == out.data_ptr()
    check(y.reshape(2 * T, 96), x.reshape(2 * T, 320), codes, packed, fmt, bias=bias)


def test_strides_alignment_and_other_orders():
    """Rows of a wider tensor, a view off 16 bytes, a transposed input, a CPU one."""
    import qwantize_b200 as q
    codes, packed = make_weight(200, 256, "nvfp4", 5)
    w = q.FP4Weight(codes, packed)
    wide = acts(70, 512 + 8, torch.bfloat16, 6).to(DEV)
    base = q.fp4_linear(wide[:, 256:512].contiguous(), w)
    assert torch.equal(q.fp4_linear(wide[:, 256:512], w), base)
    odd = torch.empty(70 * 256 + 1, dtype=torch.bfloat16, device=DEV)[1:].reshape(70, 256)
    odd.copy_(wide[:, 256:512])
    assert odd.data_ptr() % 16 and torch.equal(q.fp4_linear(odd, w), base)
    assert torch.equal(q.fp4_linear(wide[:, 256:512].T.contiguous().T, w), base)
    assert torch.equal(q.fp4_linear(wide[:, 256:512].cpu(), w), base.cpu())
    assert torch.equal(q.fp4_linear(wide[::2, 256:512], w), base[::2])
    assert torch.equal(q.fp4_linear(wide[3, 256:512], w), q.fp4_linear(wide[3:4, 256:512], w)[0])


def test_rows_of_any_magnitude():
    """The power of two of an NVFP4 row: results of a row scaled by 2^e scale by
    2^e exactly; zero rows give zeros; rows near the ends of fp32 stay finite."""
    import qwantize_b200 as q
    codes, packed = make_weight(64, 128, "nvfp4", 7)
    w = q.FP4Weight(codes, packed)
    x = acts(4, 128, torch.bfloat16, 8).float().to(DEV)
    y = q.fp4_linear(x, w)
    for e in (-60, -7, 11, 60):
        assert torch.equal(q.fp4_linear(x * 2.0**e, w), y * 2.0**e)
    x[1] = 0
    y = q.fp4_linear(x, w)
    assert not y[1].any() and bool(torch.isfinite(y).all())


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("T", [3, 150])
def test_a_row_with_a_non_finite_value_spoils_no_other(bad, T):
    import qwantize_b200 as q
    codes, packed = make_weight(40, 512, "nvfp4", 11)
    w = q.FP4Weight(codes, packed)
    x = acts(T, 512, torch.bfloat16, 12).to(DEV)
    good = q.fp4_linear(x, w)
    x[1, 200] = bad
    y = q.fp4_linear(x, w)
    assert bool(y[1].isnan().all())
    rest = [0] + list(range(2, T))
    assert torch.equal(y[rest], good[rest])


def test_same_bits_on_every_call_and_on_another_stream():
    import qwantize_b200 as q
    codes, packed = make_weight(2560, 9728, "mxfp4", 13)
    w = q.FP4Weight(codes, packed, "mxfp4")
    x = acts(48, 9728, torch.bfloat16, 14).to(DEV)
    y = q.fp4_linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [q.fp4_linear(x, w) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(y, v) for v in ys)
    check(y[:4], x[:4], codes, packed, "mxfp4")


def test_quantize_and_dequantize_a_weight():
    import qwantize_b200 as q
    g = torch.Generator().manual_seed(15)
    W = (torch.randn(96, 512, generator=g) * 0.02).to(torch.bfloat16)
    X = torch.randn(300, 512, generator=g).to(torch.bfloat16)
    for fmt in ("nvfp4", "mxfp4"):
        for method in ("naive", "optimal", "hessian"):
            w = q.FP4Weight.quantize(W.to(DEV), fmt, method, X=X.to(DEV))
            d = w.dequantize()
            assert torch.equal(d.cpu().double(), decode(w.scale_codes, w.packed, fmt, w.tensor_scale))
            # a block's largest step is a third of its largest value: far inside 0.2 of the norm
            assert float((d.cpu() - W.float()).norm() / W.float().norm()) < 0.2


def test_no_tokens():
    import qwantize_b200 as q
    codes, packed = make_weight(40, 64, "nvfp4", 1)
    assert q.fp4_linear(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), q.FP4Weight(codes, packed)).shape == (0, 40)


def test_refusals():
    import qwantize_b200 as q
    codes, packed = make_weight(40, 64, "nvfp4", 1)
    w = q.FP4Weight(codes, packed)
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (x[:, :32], x.double(), x.to(torch.int8)):
        with pytest.raises(AssertionError):
            q.fp4_linear(bad, w)
    with pytest.raises(AssertionError):
        q.fp4_linear(x, w, bias=torch.zeros(41, device=DEV))
    with pytest.raises(AssertionError):
        q.fp4_linear(x, w, out=torch.empty(2, 41, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(AssertionError):
        q.fp4_linear(x, packed)
    with pytest.raises(AssertionError):
        q.FP4Weight(codes, packed[:, :1], "nvfp4")
    with pytest.raises(AssertionError):
        q.FP4Weight(codes, packed, "mxfp4")
    with pytest.raises(AssertionError):
        q.FP4Weight(codes, packed, "int4")
