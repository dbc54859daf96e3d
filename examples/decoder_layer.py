"""A decoder layer over quantised weights and a 4-bit key / value cache: the operators of gomlx_amd.nn as a serving loop calls them.

``python examples/decoder_layer.py [--tokens N]`` takes ragged prompts through one Llama-3-8B-shaped layer (synthetic weights), decodes
N tokens of every sequence, shrinks the caches to a budget by accumulated attention weight on the way, and prints what a step takes.
"""
from __future__ import annotations

import argparse
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from gomlx_amd import ggml, nn, synth  # noqa: E402


class Layer:
    """Weights of one layer: q, k, v, o, gate, up, down as [N, bytesPerRow] blocks, with norms in front of both halves and of every
    query and key head."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, ffn: int, ggml_type: int = ggml.Q4_K, seed: int = 0, positions: int = 4096):
        self.hidden, self.heads, self.kv_heads, self.dim = hidden, heads, kv_heads, hidden // heads
        kv = kv_heads * self.dim
        shapes = dict(q=(hidden, hidden), k=(kv, hidden), v=(kv, hidden), o=(hidden, hidden), gate=(ffn, hidden), up=(ffn, hidden), down=(hidden, ffn))
        self.weights = {n: torch.from_numpy(synth.weights(ggml_type, seed + i, rows, cols)).cuda() for i, (n, (rows, cols)) in enumerate(shapes.items())}
        self.quant = nn.Quantization(ggml_type=ggml_type)
        gen = torch.Generator("cuda").manual_seed(seed)
        self.norms = [nn.RMSNorm(gain=1 + 0.1 * torch.randn(n, device="cuda", generator=gen), epsilon=1e-5) for n in (hidden, hidden, self.dim, self.dim)]
        self.cos, self.sin = nn.rotary_table(positions, self.dim, 500000.0)


class Caches:
    """Pages of one layer's keys and values, with every token's account of attention, and the sequences' page table.  Sequences hold their
    pages for good here; a server hands them out as lengths grow."""

    def __init__(self, layer: Layer, seqs: int, most: int, page_tokens: int = 64):
        self.per_seq = -(-most // page_tokens)
        self.data = nn.kv_cache(seqs * self.per_seq, layer.kv_heads, layer.dim, page_tokens)
        self.accounts = torch.zeros(seqs * self.per_seq, layer.kv_heads, page_tokens, device="cuda")
        self.table = torch.arange(seqs * self.per_seq, dtype=torch.int32, device="cuda").view(seqs, self.per_seq)
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")


def step(layer: Layer, caches: Caches, x: torch.Tensor, positions: torch.Tensor, starts: torch.Tensor | None = None, max_new: int = 1) -> torch.Tensor:
    """x: float32 [rows, hidden] of the sequences' new tokens, which ``caches.lengths`` already counts -> float32 [rows, hidden]."""
    w, q4, rows = layer.weights, layer.quant, x.shape[0]
    q, k, v = nn.quantized_dense_batch([(x, w[n], q4, None, None) for n in "qkv"], norm=layer.norms[0])
    q, k, v = q.view(rows, layer.heads, layer.dim), k.view(rows, layer.kv_heads, layer.dim), v.view(rows, layer.kv_heads, layer.dim)
    q, k = nn.qk_norm_rope(q, k, positions, layer.cos, layer.sin, q_norm=layer.norms[2], k_norm=layer.norms[3])
    nn.kv_cache_append(caches.data, k, v, caches.table, caches.lengths, starts=starts, max_new=max_new, weights=caches.accounts)
    a = nn.cached_attention(q, caches.data, caches.table, caches.lengths, starts=starts, max_new=max_new, weights=caches.accounts)
    h = nn.quantized_dense(a.view(rows, layer.hidden), w["o"], q4, residual=x)
    f = nn.gated_feed_forward(h, w["gate"], w["up"], q4, nn.Activation.SILU, norm=layer.norms[1])
    return nn.quantized_dense(f, w["down"], q4, residual=h)


def shrink(caches: Caches, keep: int, recent: int) -> None:
    """Every sequence to at most ``keep`` tokens.  Positions of new tokens go on as if nothing had left."""
    _, caches.lengths = nn.kv_cache_evict(caches.data, caches.accounts, caches.table, caches.lengths, keep, recent)


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--tokens", type=int, default=64)
    p.add_argument("--seqs", type=int, default=8)
    p.add_argument("--prompt", type=int, default=1000)
    p.add_argument("--budget", type=int, default=512)
    p.add_argument("--shape", type=int, nargs=4, default=(4096, 32, 8, 14336), metavar=("HIDDEN", "HEADS", "KV_HEADS", "FFN"))
    a = p.parse_args()
    most = a.prompt + a.tokens + 2  # (two steps warm up)
    layer = Layer(*a.shape, positions=most)
    caches = Caches(layer, a.seqs, most)
    news = [max(1, a.prompt - 37 * b) for b in range(a.seqs)]
    starts = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    caches.lengths += torch.tensor(news, dtype=torch.int32, device="cuda")
    positions = torch.cat([torch.arange(n) for n in news]).int().cuda()
    x = torch.randn(sum(news), layer.hidden, device="cuda")

    def timed(f):
        torch.cuda.synchronize()
        t = time.perf_counter()
        r = f()
        torch.cuda.synchronize()
        return r, time.perf_counter() - t

    step(layer, caches, x, positions, starts, max(news))  # (workspaces are made by the first call)
    caches.accounts.zero_()
    y, s = timed(lambda: step(layer, caches, x, positions, starts, max(news)))
    print(f"prompts of {news[-1]} to {news[0]} tokens: {1e3 * s:.2f} ms, {sum(news) / s:.0f} tokens/s a layer")
    h, position = y[starts[1:].long() - 1], torch.tensor(news, dtype=torch.int32, device="cuda")

    def decode(count):
        nonlocal h
        for _ in range(count):
            caches.lengths += 1
            h = step(layer, caches, h / h.square().mean(-1, keepdim=True).sqrt(), position)
            position.add_(1)

    decode(2)  # (as above)
    for count in (a.tokens // 2, a.tokens - a.tokens // 2):
        _, s = timed(lambda: decode(count))
        print(f"{count} tokens of {a.seqs} sequences, {caches.lengths.min().item()} to {caches.lengths.max().item()} tokens long then: {1e6 * s / max(1, count):.0f} us a step")
        _, s = timed(lambda: shrink(caches, a.budget, a.budget // 8))
        print(f"shrunk to {caches.lengths.max().item()} tokens at most: {1e6 * s:.0f} us")
    assert math.isfinite(h.abs().max().item())


if __name__ == "__main__":
    main()
