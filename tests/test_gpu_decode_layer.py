"""The serving operators together: the example's decoder layer, step by step from an
empty cache, against the same layer in fp32 on the dequantized weights.

What differs is the rounding of activations: to FP4 before the two linear products
(a value moves by at most a sixth of its block's largest, about a tenth of the row's
norm), to 8 bits in the cache, to bf16 between the operators.  The layer adds its
input twice, so its output stays within a fifth of its norm unless an operator is
wrong or a token takes another expert; most tokens are far nearer."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


def example():
    spec = importlib.util.spec_from_file_location("decode_layer", os.path.join(ROOT, "examples", "decode_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("cache", [torch.int8, torch.float8_e4m3fn])
def test_decode_layer(fmt, cache):
    ex = example()
    layer = ex.DecodeLayer(256, 8, 2, 64, experts=8, inner=128, top_k=2, fmt=fmt)
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randn(70, 5, 256, generator=g, device="cuda").to(torch.bfloat16)
    out = ex.decode(layer, tokens, cache)
    assert torch.equal(out, ex.decode(layer, tokens, cache))
    keys, values = [], []
    ref = torch.stack([layer.reference(x, keys, values) for x in tokens])
    err = (out.float() - ref).norm(dim=-1) / ref.norm(dim=-1)
    assert float(err.median()) < 0.2


def test_a_step_can_be_captured_in_a_graph():
    """No operator of a step synchronises or reads on the host: a step is captured
    once and replayed, with the same bits."""
    import qwantize_b200 as q
    ex = example()
    layer = ex.DecodeLayer(256, 8, 2, 64, experts=8, inner=128, top_k=2)
    g = torch.Generator(device="cuda").manual_seed(2)
    tokens = torch.randn(4, 3, 256, generator=g, device="cuda").to(torch.bfloat16)
    want = ex.decode(layer, tokens)
    cache = q.KVCache8(3, 2, 64)
    table = torch.arange(3, dtype=torch.int32, device="cuda").reshape(3, 1)
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")
    x = tokens[0].clone()
    layer.step(x, cache, table, lengths)  # first use sets kernel attributes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.step(x, cache, table, lengths)
    for i in range(4):
        x.copy_(tokens[i])
        lengths.fill_(i)
        graph.replay()
        assert torch.equal(y, want[i])
