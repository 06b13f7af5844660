"""What is measured of the operators that serve a quantized model.

Four operators, each in a plain form (elementary torch operations in 32 bits)
and, where ``own`` is true, through this package:

linear     y = x W^T with W in packed FP4 and x quantized to the same format on
           the way in (q.fp4_linear)
moe        a whole mixture-of-experts layer for a few tokens: router, top-k,
           gated experts in packed FP4, weighted sum (q.fp4_moe)
append     new keys and values into a paged cache held in 8 bits with one scale
           per page and head (q.kv_cache_append, read back by q.kv_cache_read)
attention  one query token per sequence over that cache (q.kv_cache_attention)

Formats: "nvfp4" is E2M1 codes with an E4M3 scale per 16 elements, "mxfp4" E2M1
codes with a power-of-two scale per 32.  Packed bytes hold element 2i in the low
nibble.  An activation row in "nvfp4" also carries a power of two t, the
smallest with max|row| <= 448 * 6 * t, so that its block scales use the E4M3
range whatever the row's magnitude."""
import math
import random

import torch

own = False

PAGE = 64  # tokens of one cache page, the block that shares a scale
BLOCK = {"nvfp4": 16, "mxfp4": 32}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}  # largest code of a cache type
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
BOUNDS = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]  # a tie takes the smaller value


def listed():
    return [
        # one token through an up projection: the smallest call of a decode step, all latency and weight bytes
        {"name": "linear 1x2560x9728", "op": "linear", "T": 1, "K": 2560, "N": 9728, "fmt": "nvfp4", "type": "bf16", "bias": False},
        # a batch of 48 sequences decoding through a down projection
        {"name": "linear 48x9728x2560 mx", "op": "linear", "T": 48, "K": 9728, "N": 2560, "fmt": "mxfp4", "type": "bf16", "bias": False},
        # a short prompt and a projection whose sizes fill no tile, with a bias
        {"name": "linear 333x2544x1000 odd", "op": "linear", "T": 333, "K": 2544, "N": 1000, "fmt": "nvfp4", "type": "f16", "bias": True},
        # an ordinary prompt
        {"name": "linear 2048x2560x9728", "op": "linear", "T": 2048, "K": 2560, "N": 9728, "fmt": "nvfp4", "type": "bf16", "bias": False},
        # a long batch of prompts through the widest projection of the 70B stack
        {"name": "linear 8192x8192x28672", "op": "linear", "T": 8192, "K": 8192, "N": 28672, "fmt": "nvfp4", "type": "bf16", "bias": False},
        # one decoded token through many small experts
        {"name": "moe 1 token 8 of 128", "op": "moe", "T": 1, "H": 2048, "I": 768, "E": 128, "top": 8, "fmt": "nvfp4", "type": "bf16"},
        # an odd batch through few experts, so that several tokens share each
        {"name": "moe 17 tokens 2 of 8 mx", "op": "moe", "T": 17, "H": 2560, "I": 1376, "E": 8, "top": 2, "fmt": "mxfp4", "type": "f16"},
        # a full decode batch: nearly every expert is read
        {"name": "moe 64 tokens 8 of 64", "op": "moe", "T": 64, "H": 2560, "I": 1280, "E": 64, "top": 8, "fmt": "nvfp4", "type": "bf16"},
        # the step of a decode batch: one token to each of 64 sequences, most inside a page that has tokens
        {"name": "append 64 x 1", "op": "append", "B": 64, "old": 500, "new": 1, "Hkv": 8, "D": 128, "cache": "int8", "type": "bf16"},
        # prompts of different lengths into the cache
        {"name": "append 8 prompts", "op": "append", "B": 8, "old": 70, "new": 1900, "Hkv": 8, "D": 128, "cache": "e4m3", "type": "f16"},
        # one short conversation
        {"name": "attention 1 x 300", "op": "attention", "B": 1, "len": 300, "Hq": 32, "Hkv": 8, "D": 128, "cache": "int8", "type": "bf16"},
        # a batch of long ones, of different lengths, an empty one among them
        {"name": "attention 32 x 32768", "op": "attention", "B": 32, "len": 32768, "Hq": 64, "Hkv": 8, "D": 128, "cache": "e4m3", "type": "bf16"},
    ]


def _spread(rng, low, high, step=1):
    return max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))) // step * step))


def draw(rng):
    op = rng.choice(["linear", "linear", "moe", "moe", "append", "attention", "attention"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    kind = rng.choice(["bf16", "f16"])
    if op == "linear":
        T = _spread(rng, 1, 8192)
        return {"op": op, "T": T, "K": _spread(rng, 256, 9728, BLOCK[fmt]), "N": _spread(rng, 96, 28672), "fmt": fmt, "type": kind,
                "bias": rng.random() < 0.5}
    if op == "moe":
        E = rng.choice([4, 8, 13, 32, 64, 128])
        H, I = _spread(rng, 256, 2560, 32), _spread(rng, 96, 1280, 32)
        while E * H * I > 64 * 2560 * 1280:
            E //= 2
        return {"op": op, "T": _spread(rng, 1, 64), "H": H, "I": I, "E": E, "top": rng.randint(1, min(8, E)), "fmt": fmt, "type": kind}
    Hkv, D, cache = rng.choice([1, 2, 4, 8]), rng.choice([64, 128]), rng.choice(["int8", "e4m3"])
    if op == "append":
        return {"op": op, "B": _spread(rng, 1, 64), "old": _spread(rng, 1, 1000), "new": rng.choice([1, 1, _spread(rng, 2, 300)]), "Hkv": Hkv, "D": D,
                "cache": cache, "type": kind}
    B = _spread(rng, 1, 64)
    return {"op": op, "B": B, "len": _spread(rng, 1, min(32768, 600000 // B)), "Hq": Hkv * rng.choice([1, 2, 4, 5, 8, 16]), "Hkv": Hkv, "D": D,
            "cache": cache, "type": kind}


# --- the formats, in 32 or 64 bits -------------------------------------------


def _power(amax):
    """The smallest power of two t with amax <= 2688 t (1 for 0 and what is not finite)."""
    m, e = torch.frexp(amax)
    p = torch.where(m <= 0.65625, e - 12, e - 11).clamp(min=-120)
    t = torch.ldexp(torch.ones_like(amax), p)
    return torch.where((amax > 0) & torch.isfinite(amax), t, torch.ones_like(amax))


def _quantize(y, fmt):
    """Rows of y (..., K) in blocks: the scale of each and the codes (0..15), in y's precision."""
    b = y.reshape(*y.shape[:-1], -1, BLOCK[fmt])
    amax = b.abs().amax(-1)
    if fmt == "nvfp4":
        scale = (amax / 6).float().to(torch.float8_e4m3fn).to(y.dtype)
    else:
        scale = torch.ldexp(torch.ones_like(amax), (torch.frexp(amax.clamp(min=1e-30))[1] - 3).clamp(-126, 127))
    bounds = torch.tensor(BOUNDS, dtype=y.dtype, device=y.device)
    over = b.abs() / scale.unsqueeze(-1)
    code = torch.bucketize(torch.where(scale.unsqueeze(-1) > 0, over, torch.zeros_like(over)), bounds)
    return scale, code + 8 * (b < 0)


def _dequantize(scale, code, dtype=torch.float32):
    values = torch.tensor(VALUES, dtype=dtype, device=code.device)
    return (values[code] * scale.unsqueeze(-1)).flatten(-2)


def _unpack(w, fmt, dtype=torch.float32):
    """The values of a packed weight: scale bytes (..., K / block), packed (..., K / 2), and its tensor scale."""
    codes, packed, t = w
    scale = codes.view(torch.float8_e4m3fn).to(dtype) if fmt == "nvfp4" else torch.ldexp(torch.ones_like(codes, dtype=dtype), codes.int() - 127)
    nibbles = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).int()
    return _dequantize(scale * t, nibbles.reshape(*codes.shape, -1), dtype)


def _rows(x, fmt, dtype=torch.float32):
    """Activation rows as the values that their FP4 form stands for."""
    x = x.to(dtype)
    t = _power(x.abs().amax(-1, keepdim=True)) if fmt == "nvfp4" else torch.ones_like(x[..., :1])
    return _dequantize(*_quantize(x / t, fmt), dtype) * t


# --- inputs --------------------------------------------------------------------


def _weight(g, N, K, fmt):
    """A packed weight as it is stored: normal values with a few outliers, on one tensor scale."""
    w = torch.randn(N, K, generator=g, device="cuda") * (1 / math.sqrt(K))
    w = torch.where(torch.rand(N, K, generator=g, device="cuda") < 1e-3, w * 8, w)
    t = 2.0**-9 if fmt == "nvfp4" else 1.0
    scale, code = _quantize((w / t).clamp(-2600, 2600), fmt)
    code = code.flatten(-2)
    packed = (code[..., ::2] + 16 * code[..., 1::2]).to(torch.uint8)
    codes = scale.to(torch.float8_e4m3fn).view(torch.uint8) if fmt == "nvfp4" else (torch.frexp(scale)[1] + 126).to(torch.uint8)
    return codes, packed, t


def _weights(g, E, N, K, fmt):
    parts = [_weight(g, N, K, fmt) for _ in range(E)]
    return torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts]), parts[0][2]


def _lengths(B, most, empty):
    """B lengths from 1 to `most`, of the sizes alone, so that another seed's outputs have the same shapes."""
    r = random.Random("%d %d" % (B, most))
    n = [most] + [max(1, int(most * r.uniform(0.1, 1.0))) for _ in range(B - 1)]
    if empty and B > 2:
        n[B // 2] = 0
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, op = case, case["op"]
    kind = TYPES[c["type"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    if own:
        import qwantize_b200 as q
    if op == "linear":
        s = {"x": (normal(c["T"], c["K"]) * torch.exp(normal(c["K"]))).to(kind), "w": _weight(g, c["N"], c["K"], c["fmt"]),
             "bias": normal(c["N"]).to(kind) if c["bias"] else None}
        if own:
            s["weight"] = q.FP4Weight(s["w"][0], s["w"][1], c["fmt"], tensor_scale=s["w"][2])
    elif op == "moe":
        s = {"x": normal(c["T"], c["H"]).to(kind), "router": (normal(c["E"], c["H"]) * (2 / math.sqrt(c["H"]))).to(kind),
             "up": _weights(g, c["E"], 2 * c["I"], c["H"], c["fmt"]), "down": _weights(g, c["E"], c["H"], c["I"], c["fmt"])}
        if own:
            s["experts"] = q.FP4Experts(s["up"][:2], s["down"][:2], c["fmt"], tensor_scales=(s["up"][2], s["down"][2]))
    else:
        B, Hkv, D, new = c["B"], c["Hkv"], c["D"], c.get("new", 0)
        old = _lengths(B, c.get("len", c.get("old")), op == "attention")
        pages = -(-(int(old.max()) + new) // PAGE)  # of the longest sequence: the width of the block table
        table = torch.randperm(B * pages, generator=g, device="cuda").int().reshape(B, pages)
        k, v = (normal(B * pages, Hkv, 1, D).mul(0.5).exp() * normal(B * pages, Hkv, PAGE, D) for _ in range(2))
        (kc, ks), (vc, vs) = _to8(k, c["cache"]), _to8(v, c["cache"])
        s = {"table": table, "old": old, "k": kc, "ks": ks, "v": vc, "vs": vs}
        if op == "attention":
            s["q"] = normal(B, c["Hq"], D).to(kind)
        else:
            take = _lengths(B, new, False)
            s["cu"] = torch.nn.functional.pad(take.cumsum(0), (1, 0)).int()
            s["most"] = int(take.max())
            total = int(s["cu"][-1])
            s["nk"], s["nv"] = ((normal(total, Hkv, 1).exp() * normal(total, Hkv, D)).to(kind) for _ in range(2))
            seq = torch.repeat_interleave(torch.arange(B, device="cuda"), take)
            at = torch.arange(total, device="cuda") - s["cu"][seq] + old[seq]
            s["page"], s["slot"] = table[seq, at // PAGE].long(), at % PAGE  # where each new token goes
            s["touched"] = torch.unique(s["page"]).int()
            # slots that hold tokens already; what lies behind them in a page is of no sequence
            held = (torch.arange(pages * PAGE, device="cuda") < old[:, None]).reshape(B, pages, PAGE)
            s["held"] = torch.zeros(B * pages, PAGE, dtype=torch.bool, device="cuda")
            s["held"][table.long()] = held
        if own:
            s["cache"] = q.KVCache8(B * pages, Hkv, D, TYPES[c["cache"]], device="cuda")
            s["cache"].load_codes(s["k"], s["ks"], s["v"], s["vs"])
    return {**s, "case": dict(case)}


def _to8(x, cache):
    """Pages (..., PAGE, D) in 8 bits with one scale each."""
    scale = x.abs().amax((-1, -2)) / TOP[cache]
    return _code8(x / scale[..., None, None], cache), scale


def _code8(y, cache):
    return y.round().clamp(-127, 127).to(torch.int8) if cache == "int8" else y.clamp(-448, 448).float().to(torch.float8_e4m3fn)


# --- one pass ------------------------------------------------------------------


def run(state):
    return (_own if own else _plain)[state["case"]["op"]](state)


def _own_linear(s):
    import qwantize_b200 as q

    return q.fp4_linear(s["x"], s["weight"], bias=s["bias"])


def _own_moe(s):
    import qwantize_b200 as q

    y, ids, weights = q.fp4_moe(s["x"], s["router"], s["experts"], s["case"]["top"], return_routing=True)
    return {"y": y, "ids": ids, "weights": weights}


def _own_append(s):
    import qwantize_b200 as q

    q.kv_cache_append(s["cache"], s["nk"], s["nv"], s["table"], s["old"], cu_new=s["cu"], max_new=s["most"])
    k, v = q.kv_cache_read(s["cache"], s["touched"])
    return {"k": k, "v": v}


def _own_attention(s):
    import qwantize_b200 as q

    return q.kv_cache_attention(s["cache"], s["q"], s["table"], s["old"])


def _plain_linear(s):
    fmt = s["case"]["fmt"]
    y = _rows(s["x"], fmt) @ _unpack(s["w"], fmt).T
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)


def _route(x, router, top):
    logits = x @ router.T
    order = torch.sort(logits, dim=-1, descending=True, stable=True)  # a tie takes the lower index
    ids = order.indices[:, :top]
    return ids.int(), torch.softmax(order.values[:, :top], -1)


def _plain_moe(s):
    c = s["case"]
    x = s["x"].float()
    ids, weights = _route(x, s["router"].float(), c["top"])
    h = x[None] @ _unpack(s["up"], c["fmt"]).transpose(1, 2)  # every expert for every token: (E, T, 2 I)
    gate, up = h[..., : c["I"]], h[..., c["I"] :]
    y = (gate / (1 + torch.exp(-gate)) * up) @ _unpack(s["down"], c["fmt"]).transpose(1, 2)
    share = torch.zeros(c["T"], c["E"], device=x.device).scatter(1, ids.long(), weights)
    return {"y": (share.T[..., None] * y).sum(0).to(s["x"].dtype), "ids": ids, "weights": weights}


def _appended(s, k, ks, new, dtype):
    """Pages of one of the two halves after the append: a page's scale grows to what its new tokens need, and
    its codes are then taken over to the larger scale; a page without tokens starts from nothing."""
    cache, touched = s["case"]["cache"], s["touched"].long()
    new = new.to(dtype)
    held = s["held"]
    largest = torch.full(ks.shape, 0.0, dtype=dtype, device=ks.device).index_reduce(0, s["page"], new.abs().amax(-1), "amax")
    before = torch.where(held.any(-1)[:, None], ks.to(dtype), torch.zeros_like(largest))
    scale = torch.maximum(before, largest / TOP[cache])[touched]
    before = before[touched]
    ratio = torch.where(scale > 0, before / scale, torch.zeros_like(scale))[..., None, None]
    codes = _code8(torch.where(held[touched][:, None, :, None], k[touched].to(dtype), torch.zeros((), dtype=dtype, device=ks.device)) * ratio, cache)
    place = torch.full((k.shape[0],), 0, dtype=torch.long, device=ks.device).scatter(0, touched, torch.arange(len(touched), device=ks.device))
    at = place[s["page"]]
    over = torch.where(scale[at][..., None] > 0, new / scale[at][..., None], torch.zeros_like(new))
    codes.transpose(1, 2)[at, s["slot"]] = _code8(over, cache)
    return codes, scale


def _plain_append(s):
    out, touched = {}, s["touched"].long()
    for name, codes, scales, new in (("k", "k", "ks", "nk"), ("v", "v", "vs", "nv")):
        c, t = _appended(s, s[codes], s[scales], s[new], torch.float32)
        s[codes][touched], s[scales][touched] = c, t
        out[name] = c.float() * t[..., None, None]
    return out


def _attend(s, dtype):
    c, n = s["case"], s["old"]
    table = s["table"].long()
    flat = lambda codes, scale: (codes[table].to(dtype) * scale[table][..., None, None].to(dtype)).transpose(1, 2).flatten(2, 3)  # noqa: E731
    B, G = c["B"], c["Hq"] // c["Hkv"]
    q = s["q"].to(dtype).reshape(B, c["Hkv"], G, c["D"])
    a = q @ flat(s["k"], s["ks"]).transpose(2, 3) / math.sqrt(c["D"])  # (B, Hkv, G, tokens)
    away = (torch.arange(a.shape[-1], device=a.device) >= n[:, None])[:, None, None]
    a = a.masked_fill(away, -math.inf)
    top = a.amax(-1, keepdim=True).clamp(min=torch.finfo(dtype).min)
    e = torch.exp(a - top)
    total = e.sum(-1, keepdim=True)
    y = e @ flat(s["v"], s["vs"]) / torch.where(total > 0, total, torch.ones_like(total))  # an empty sequence gives zeros
    return y.reshape(B, c["Hq"], c["D"])


def _plain_attention(s):
    return _attend(s, torch.float32).to(s["q"].dtype)


_own = {"linear": _own_linear, "moe": _own_moe, "append": _own_append, "attention": _own_attention}
_plain = {"linear": _plain_linear, "moe": _plain_moe, "append": _plain_append, "attention": _plain_attention}


# --- 64 bits -------------------------------------------------------------------

_E2M1 = [(-1) ** (i >> 3) * (i & 1) / 2 if not i >> 1 & 3 else (-1) ** (i >> 3) * 2.0 ** ((i >> 1 & 3) - 1) * (1 + (i & 1) / 2) for i in range(16)]


def _two(e):
    """2^e in 64 bits from its bits, exact where a power function need not be."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _decode64(w, fmt):
    """A packed weight by the definition of its bytes."""
    codes, packed, t = w
    c = codes.double()
    if fmt == "nvfp4":
        e, m = torch.div(c, 8, rounding_mode="floor"), c % 8
        scale = torch.where(e > 0, _two(e - 7) * (1 + m / 8), m * 2.0**-9)
    else:
        scale = _two(c - 127)
    table = torch.tensor(_E2M1, dtype=torch.float64, device=c.device)
    v = torch.empty(*packed.shape, 2, dtype=torch.float64, device=c.device)
    v[..., 0], v[..., 1] = table[(packed % 16).long()], table[torch.div(packed, 16, rounding_mode="floor").long()]
    return v.reshape(*codes.shape, -1).mul_(scale[..., None] * t).flatten(-2)


def _nearest64(x, fmt):
    """Activation rows as FP4 values by the definition: the nearest of the eight magnitudes, a tie to the smaller."""
    x = x.double()
    t = torch.ones_like(x[:, :1])
    if fmt == "nvfp4":
        amax = x.abs().amax(-1, keepdim=True)
        m, e = torch.frexp(amax / 2688)
        t = torch.where(amax > 0, _two(torch.where(m == 0.5, e - 1, e)), t)
    b = (x / t).reshape(x.shape[0], -1, BLOCK[fmt])
    amax = b.abs().amax(-1, keepdim=True)
    if fmt == "nvfp4":
        ulp = _two(torch.frexp((amax / 6).clamp(min=2.0**-6))[1] - 4)
        scale = torch.round(amax / 6 / ulp) * ulp  # half to even
    else:
        scale = _two(torch.frexp(amax.clamp(min=1e-30))[1] - 3)
    a = b.abs() / torch.where(scale > 0, scale, torch.ones_like(scale))
    q = torch.zeros_like(a)
    for low, high in zip(_E2M1[:7], _E2M1[1:8]):
        q = torch.where(a > (low + high) / 2, torch.full_like(q, high), q)
    return (torch.sign(b) * q * scale).reshape(x.shape) * t


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "linear":
        w, x = _decode64(s["w"], case["fmt"]), _nearest64(s["x"], case["fmt"])
        y = x @ w.T
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "moe":
        x = s["x"].double()
        logits = x @ s["router"].double().T
        values, ids = torch.topk(logits, case["top"], dim=-1)
        weights = torch.exp(values - values[:, :1])
        weights = weights / weights.sum(-1, keepdim=True)
        y = torch.zeros_like(x)
        for e in range(case["E"]):
            rows, nth = torch.nonzero(ids == e, as_tuple=True)
            if not len(rows):
                continue
            h = x[rows] @ _decode64((s["up"][0][e], s["up"][1][e], s["up"][2]), case["fmt"]).T
            gate, up = h[:, : case["I"]], h[:, case["I"] :]
            out = (gate * torch.sigmoid(gate) * up) @ _decode64((s["down"][0][e], s["down"][1][e], s["down"][2]), case["fmt"]).T
            y[rows] += weights[rows, nth, None] * out
        return {"y": y, "ids": None, "weights": weights}
    if op == "append":
        out, top = {}, TOP[case["cache"]]
        for name, codes, scales, new in (("k", "k", "ks", "nk"), ("v", "v", "vs", "nv")):
            c, t = _appended(s, s[codes], s[scales], s[new], torch.float64)
            out[name] = c.double() * t[..., None, None]
        return out
    if case["B"] * case["len"] * case["Hkv"] > 32 * 32768 * 8:
        return None
    out = []
    for b in range(case["B"]):  # one sequence at a time, its own tokens alone
        n = int(s["old"][b])
        pages = s["table"][b, : -(-n // PAGE)].long()
        k, v = ((s[c][pages].double() * s[t][pages].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n] for c, t in (("k", "ks"), ("v", "vs")))
        q = s["q"][b].double().reshape(case["Hkv"], -1, case["D"])
        out.append((torch.softmax(q @ k.transpose(1, 2) * case["D"] ** -0.5, -1) @ v).reshape(case["Hq"], case["D"]))
    return torch.stack(out)


def work(case):
    c, op = case, case["op"]
    per = {"nvfp4": 0.5 + 1 / 16, "mxfp4": 0.5 + 1 / 32}  # bytes of one stored weight
    if op == "linear":
        T, K, N = c["T"], c["K"], c["N"]
        return {"bytes": N * K * per[c["fmt"]] + 2 * T * K + 2 * T * N + (2 * N if c["bias"] else 0), "flops": 2 * T * K * N}
    if op == "moe":
        T, H, I, E, top = c["T"], c["H"], c["I"], c["E"], c["top"]
        read = E * (1 - (1 - top / E) ** T)  # experts that some token takes, for evenly spread choices
        return {"bytes": read * 3 * H * I * per[c["fmt"]] + 2 * E * H + 4 * T * H, "flops": T * top * 6 * H * I + 2 * T * E * H}
    row = c["Hkv"] * c["D"]
    if op == "append":
        tokens = c["B"] * max(1, 0.55 * c["new"])
        pages = c["B"] * (1 + max(1, 0.55 * c["new"]) / PAGE)
        return {"bytes": 2 * row * (tokens * (2 + 1) + pages * PAGE * (1 + 4)), "flops": 8 * row * tokens}
    tokens = 0.55 * c["B"] * c["len"]
    return {"bytes": 2 * row * tokens + 4 * c["B"] * c["Hq"] * c["D"], "flops": 4 * tokens * c["Hq"] * c["D"]}
