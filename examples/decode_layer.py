"""One decoder layer of a quantized mixture-of-experts model, a decode step at a time.

    python examples/decode_layer.py [--batch 8] [--steps 100] [--fmt nvfp4] [--cache int8]

Every weight matrix is NVFP4 or MXFP4 as this package quantizes it, keys and values
are kept in 8 bits, and a step is the package's serving operators with RMS norms
and residual additions between them:

    qkv   = fp4_linear(norm(x))                  packed weight, activations quantized on the way in
    kv_cache_append(k, v)                        8-bit pages, one scale per page and head
    x    += fp4_linear(kv_cache_attention(q))    grouped heads
    x    += fp4_moe(norm(x))                     router, top-k, gated experts, weighted sum

It prints the time of a step and how far the layer's output is from the same layer
with its weights dequantized and everything else in fp32."""
from __future__ import annotations

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..")))

import qwantize_b200 as q  # noqa: E402


def rms_norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class DecodeLayer:
    """hidden -> hidden with `heads` query heads on `kv_heads` cache heads of
    `head_dim`, and `experts` gated experts of width `inner`, `top_k` per token."""

    def __init__(self, hidden, heads, kv_heads, head_dim, experts, inner, top_k, fmt="nvfp4", method="optimal", seed=0,
                 dtype=torch.bfloat16, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.top_k = heads, kv_heads, head_dim, top_k

        def weight(*shape):
            return (torch.randn(*shape, generator=g, device=device) / math.sqrt(shape[-1])).to(dtype)

        self.qkv = q.FP4Weight.quantize(weight((heads + 2 * kv_heads) * head_dim, hidden), fmt, method)
        self.out = q.FP4Weight.quantize(weight(hidden, heads * head_dim), fmt, method)
        self.router = weight(experts, hidden)
        up, down = weight(experts, 2 * inner, hidden), weight(experts, hidden, inner)
        self.experts = q.FP4Experts.quantize(up, down, fmt, method)
        # what the experts' packed weights stand for, for reference() alone
        self._experts = [q.FP4Weight.quantize(w.reshape(-1, w.shape[-1]), fmt, method).dequantize().reshape(w.shape) for w in (up, down)]

    def step(self, x, cache, table, lengths):
        """x (batch, hidden) of one new token per sequence -> (batch, hidden); the
        token's key and value go into the cache at position lengths[b]."""
        B, H, K, D = x.shape[0], self.heads, self.kv_heads, self.head_dim
        qkv = q.fp4_linear(rms_norm(x), self.qkv).reshape(B, H + 2 * K, D)
        q.kv_cache_append(cache, qkv[:, H:H + K], qkv[:, H + K:], table, lengths)
        a = q.kv_cache_attention(cache, qkv[:, :H], table, lengths + 1)
        x = x + q.fp4_linear(a.reshape(B, H * D), self.out)
        return x + q.fp4_moe(rms_norm(x), self.router, self.experts, self.top_k)

    def reference(self, x, keys, values):
        """The same step in fp32 on the dequantized weights, with plain lists of the
        sequences' keys and values (B, kv_heads, D) per token."""
        B, H, K, D = x.shape[0], self.heads, self.kv_heads, self.head_dim
        x = x.float()
        qkv = (rms_norm(x) @ self.qkv.dequantize().T).reshape(B, H + 2 * K, D)
        keys.append(qkv[:, H:H + K])
        values.append(qkv[:, H + K:])
        k, v = torch.stack(keys, 2), torch.stack(values, 2)
        s = qkv[:, :H].reshape(B, K, H // K, D) @ k.transpose(2, 3) / math.sqrt(D)
        a = (torch.softmax(s, -1) @ v).reshape(B, H * D)
        x = x + a @ self.out.dequantize().T
        h = rms_norm(x)
        logits, ids = torch.topk(h @ self.router.float().T, self.top_k, dim=-1)
        share = torch.softmax(logits, -1)
        up, down = self._experts
        y = torch.zeros_like(x)
        for n in range(self.top_k):
            gate, lin = (up[ids[:, n]] @ h[..., None])[..., 0].chunk(2, -1)
            y += share[:, n, None] * (down[ids[:, n]] @ (torch.nn.functional.silu(gate) * lin)[..., None])[..., 0]
        return x + y


def decode(layer, tokens, cache_dtype=torch.int8):
    """Run tokens (steps, batch, hidden) through the layer from an empty cache:
    the outputs of all steps."""
    steps, B, _ = tokens.shape
    pages = -(-steps // q.KVCache8.page)
    cache = q.KVCache8(B * pages, layer.kv_heads, layer.head_dim, cache_dtype, device=tokens.device)
    table = torch.arange(B * pages, dtype=torch.int32, device=tokens.device).reshape(B, pages)
    lengths = torch.zeros(B, dtype=torch.int32, device=tokens.device)
    out = []
    for x in tokens:
        out.append(layer.step(x, cache, table, lengths))
        lengths += 1
    return torch.stack(out)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--fmt", choices=("nvfp4", "mxfp4"), default="nvfp4")
    ap.add_argument("--cache", choices=("int8", "e4m3"), default="int8")
    a = ap.parse_args()
    layer = DecodeLayer(2560, 32, 8, 128, experts=32, inner=768, top_k=4, fmt=a.fmt)
    tokens = torch.randn(a.steps, a.batch, 2560, device="cuda").to(torch.bfloat16)
    kind = torch.int8 if a.cache == "int8" else torch.float8_e4m3fn
    out = decode(layer, tokens, kind)
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    decode(layer, tokens, kind)
    end.record()
    torch.cuda.synchronize()
    keys, values = [], []
    ref = torch.stack([layer.reference(x, keys, values) for x in tokens])
    print(f"{a.fmt} weights, {a.cache} cache, batch {a.batch}: {begin.elapsed_time(end) / a.steps * 1e3:.0f} us a step, "
          f"{float((out.float() - ref).norm() / ref.norm()):.3f} from the fp32 layer on the dequantized weights")


if __name__ == "__main__":
    main()
