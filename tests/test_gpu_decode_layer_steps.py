"""Every operator call of the example's decoder layer against its definition in 64
bits, on the inputs that it got, and what passes between the calls, bit for bit.

Each token of each sequence is held to the operators' own bounds (the oracles of
their tests) at every step, past a page's end too: nothing is left to a median."""
import pytest
import torch

from tests import test_gpu_kv_cache, test_gpu_linear, test_gpu_moe
from tests.test_gpu_decode_layer import example
from tests.test_gpu_linear import ROUND

pytestmark = pytest.mark.gpu
STEPS, B, HIDDEN, HEADS, KV, D, TOP = 70, 5, 256, 8, 2, 64, 2


def norm(x):
    """The layer's norm in 64 bits, and the bound of its fp32 form rounded to bf16."""
    f = x.cpu().double()
    y = f / (f.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    return y, (ROUND[x.dtype] + 600 * 2.0**-24) * y.abs()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
def test_every_call_of_every_step(fmt, kind, monkeypatch):
    import qwantize_b200 as q
    ex = example()
    layer = ex.DecodeLayer(HIDDEN, HEADS, KV, D, experts=8, inner=128, top_k=TOP, fmt=fmt)
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randn(STEPS, B, HIDDEN, generator=g, device="cuda").to(torch.bfloat16)
    calls = []

    def spy(name):
        real = getattr(q, name)

        def call(*args, **kwargs):
            before = args[0].codes() if name == "kv_cache_append" else None
            got = [a.clone() if torch.is_tensor(a) else a for a in args]
            out = real(*args, **kwargs)
            after = args[0].codes() if name.startswith("kv") else None
            calls.append((name, got, out, before, after))
            return out

        monkeypatch.setattr(q, name, call)

    operators = ("fp4_linear", "kv_cache_append", "kv_cache_attention", "fp4_linear", "fp4_moe")
    moe = q.fp4_moe
    for name in dict.fromkeys(operators):
        spy(name)
    out = ex.decode(layer, tokens, kind)
    monkeypatch.undo()
    assert [c[0] for c in calls] == list(operators) * STEPS
    # the oracle of the expert layer on the values that its weights stand for
    monkeypatch.setattr(test_gpu_moe, "decode", lambda values, *_: values.cpu().double())
    for i, x in enumerate(tokens):
        (_, (h, w1), qkv, *_), (_, (cache, k, v, table, n), _, before, after), (_, (_, query, t2, n2), a, _, seen), \
            (_, (a2, w2), o, *_), (_, (m, router, experts, top), y, *_) = calls[5 * i: 5 * i + 5]
        assert w1 is layer.qkv and w2 is layer.out and experts is layer.experts and torch.equal(router, layer.router) and top == TOP
        # between the calls
        for given, of in ((h, x), (m, x + o)):
            ref, lim = norm(of)
            assert bool(((given.cpu().double() - ref).abs() <= lim).all())
        rows = qkv.reshape(B, HEADS + 2 * KV, D)
        assert torch.equal(query, rows[:, :HEADS]) and torch.equal(k, rows[:, HEADS: HEADS + KV]) and torch.equal(v, rows[:, HEADS + KV:])
        assert n.tolist() == [i] * B and n2.tolist() == [i + 1] * B and torch.equal(table, t2)
        assert torch.equal(a2, a.reshape(B, HEADS * D)) and torch.equal(out[i], x + o + y)
        # the calls
        for given, w, got in ((h, w1, qkv), (a2, w2, o)):
            test_gpu_linear.check(got, given, w.scale_codes, w.packed[:, : w.K // 2], fmt, w.tensor_scale)
        for j, new in ((0, k), (2, v)):
            codes, scale = test_gpu_kv_cache.appended(before[j].cpu(), before[j + 1].cpu(), new.cpu(), table.cpu(), [i] * B, [1] * B, kind)
            assert torch.equal(after[j].cpu().float(), codes.float()) and torch.equal(after[j + 1].cpu(), scale)
            assert torch.equal(seen[j].view(torch.uint8), after[j].view(torch.uint8)) and torch.equal(seen[j + 1], after[j + 1])
        test_gpu_kv_cache.check(a, query, *(s.cpu() for s in seen), table, n2)
        again, ids, _ = moe(m, router, experts, TOP, return_routing=True)
        assert torch.equal(again, y)
        ref, err, _, _, logits, el = test_gpu_moe.oracle(m, router, (layer._experts[0],) * 2, (layer._experts[1],) * 2, fmt, 1.0, TOP, True, ids)
        best = logits.topk(TOP, dim=-1).values
        assert bool(((logits.gather(1, ids.cpu().long()) - best).abs() <= 2 * el.amax(-1, keepdim=True)).all())
        assert bool(((y.cpu().double() - ref).abs() <= err + ROUND[y.dtype] * (ref.abs() + err) + 1e-30).all())
