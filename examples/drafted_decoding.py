"""Decoding with drafted tokens: the operators of gomlx_amd.nn as a serving loop with speculation calls them.

``python examples/drafted_decoding.py [--steps N]`` takes prompts through one Llama-3-8B-shaped layer (synthetic weights) between a token table and an
output head, then decodes: a cheap guess (the layer without its attention) drafts a tree of continuations of every sequence, one pass takes all of them through the layer over
its 4-bit cache, a token is sampled behind each of them, and the path that the samples follow is kept.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path[:0] = [os.path.dirname(os.path.abspath(__file__)), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))]
from decoder_layer import Caches, Layer  # noqa: E402
from gomlx_amd import ggml, nn, synth  # noqa: E402


class Model:
    """A layer between a token table and an output head, both [vocab, bytesPerRow]."""

    def __init__(self, vocab: int, *shape, seed: int = 0, positions: int = 4096):
        self.layer = Layer(*shape, seed=seed, positions=positions)
        self.quant = nn.Quantization(ggml_type=ggml.Q8_0)
        self.table, self.head = (torch.from_numpy(synth.weights(ggml.Q8_0, seed + 50 + i, vocab, self.layer.hidden)).cuda() for i in range(2))

    def embed(self, tokens: torch.Tensor) -> torch.Tensor:
        x = nn.quantized_gather(self.table, tokens[:, None], self.quant)
        return 512.0 * nn.rms_norm(x, nn.RMSNorm())  # (large beside what attention over random keys adds, so that the cheap guess is a good one)

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        return nn.quantized_dense(x, self.head, self.quant, norm=nn.RMSNorm())

    def feed_forward(self, h: torch.Tensor) -> torch.Tensor:
        w, q4 = self.layer.weights, self.layer.quant
        f = nn.gated_feed_forward(h, w["gate"], w["up"], q4, nn.Activation.SILU, norm=self.layer.norms[1])
        return nn.quantized_dense(f, w["down"], q4, residual=h)

    def guess(self, tokens: torch.Tensor) -> torch.Tensor:
        return self.logits(self.feed_forward(self.embed(tokens)))

    def forward(self, caches: Caches, tokens, positions, lengths, starts, max_new, tree=None) -> torch.Tensor:
        """float32 [rows, hidden] of the sequences' new tokens, which ``lengths`` counts; with ``tree`` they are drafted ones."""
        layer, rows, x = self.layer, tokens.shape[0], self.embed(tokens)
        w, q4 = layer.weights, layer.quant
        q, k, v = nn.quantized_dense_batch([(x, w[n], q4, None, None) for n in "qkv"], norm=layer.norms[0])
        q, k, v = q.view(rows, layer.heads, layer.dim), k.view(rows, layer.kv_heads, layer.dim), v.view(rows, layer.kv_heads, layer.dim)
        q, k = nn.qk_norm_rope(q, k, positions, layer.cos, layer.sin, q_norm=layer.norms[2], k_norm=layer.norms[3])
        nn.kv_cache_append(caches.data, k, v, caches.table, lengths, starts=starts, max_new=max_new)
        if tree is None:
            a = nn.cached_attention(q, caches.data, caches.table, lengths, starts=starts, max_new=max_new)
        else:
            a = nn.tree_attention(q, caches.data, caches.table, lengths, tree, starts=starts, max_new=max_new)
        return self.feed_forward(nn.quantized_dense(a.view(rows, layer.hidden), w["o"], q4, residual=x))


class Drafts:
    """Trees of one shape for every sequence: ``widths[d]`` children of every node of depth d, nodes level by level."""

    def __init__(self, seqs: int, widths):
        parents, level = [-1], [0]
        for width in widths:
            level = [len(parents) + i for i in range(len(level) * width)]
            parents += [p for p in range(level[0] - len(level) // width, level[0]) for _ in range(width)]
        self.widths, self.nodes = tuple(widths), len(parents)
        self.parents = torch.tensor(parents * seqs, dtype=torch.int32, device="cuda")
        self.starts = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * self.nodes

    def draft(self, model: Model, roots: torch.Tensor) -> torch.Tensor:
        """int32 [sequences * nodes]: under each node the likeliest tokens by the guess."""
        levels = [roots[:, None]]
        for width in self.widths:
            best = model.guess(levels[-1].reshape(-1)).topk(width).indices
            levels.append(best.int().view(len(roots), -1))
        return torch.cat(levels, 1).reshape(-1)


def step(model: Model, caches: Caches, drafts: Drafts, roots: torch.Tensor, uniform: torch.Tensor, **how) -> tuple:
    """One step of every sequence, whose last sampled tokens are ``roots`` (not yet in the cache) -> (path, next roots); ``caches.lengths`` moves on."""
    tokens = drafts.draft(model, roots)
    tree, positions = nn.draft_tree(drafts.parents, caches.lengths, starts=drafts.starts, max_new=drafts.nodes)
    lengths = caches.lengths + drafts.nodes
    h = model.forward(caches, tokens, positions, lengths, drafts.starts, drafts.nodes, tree)
    sampled = nn.sample(model.logits(h), uniform, **how)
    path, roots, caches.lengths = nn.kv_cache_accept(caches.data, caches.table, lengths, drafts.parents, tokens, sampled, starts=drafts.starts, max_new=drafts.nodes)
    return path, roots


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__)
    p.add_argument("--steps", type=int, default=32)
    p.add_argument("--seqs", type=int, default=4)
    p.add_argument("--prompt", type=int, default=500)
    p.add_argument("--vocab", type=int, default=32000)
    p.add_argument("--widths", type=int, nargs="+", default=(3, 2, 1))
    p.add_argument("--temperature", type=float, default=0.05)
    p.add_argument("--shape", type=int, nargs=4, default=(4096, 32, 8, 14336), metavar=("HIDDEN", "HEADS", "KV_HEADS", "FFN"))
    a = p.parse_args()
    drafts = Drafts(a.seqs, a.widths)
    most = a.prompt + (a.steps + 2) * (len(a.widths) + 1) + drafts.nodes
    model = Model(a.vocab, *a.shape, positions=most)
    caches = Caches(model.layer, a.seqs, most)
    starts = torch.arange(a.seqs + 1, dtype=torch.int32, device="cuda") * a.prompt
    caches.lengths += a.prompt
    tokens = torch.randint(a.vocab, (a.seqs * a.prompt,), dtype=torch.int32, device="cuda")
    h = model.forward(caches, tokens, torch.arange(a.prompt, dtype=torch.int32, device="cuda").repeat(a.seqs), caches.lengths, starts, a.prompt)
    how = dict(temperature=a.temperature, top_k=50, top_p=0.95)
    roots = nn.sample(model.logits(h[starts[1:].long() - 1]), torch.rand(a.seqs, device="cuda"), **how)
    kept = 0
    for i in range(a.steps + 2):
        if i == 2:  # (two steps warm up)
            torch.cuda.synchronize()
            before, t = caches.lengths.sum().item(), time.perf_counter()
        path, roots = step(model, caches, drafts, roots, torch.rand(a.seqs * drafts.nodes, device="cuda"), **how)
    torch.cuda.synchronize()
    t, kept = time.perf_counter() - t, caches.lengths.sum().item() - before
    print(f"{a.steps} steps of {a.seqs} sequences, {drafts.nodes} nodes each: {1e6 * t / a.steps:.0f} us a step, {kept / a.steps / a.seqs:.2f} tokens a sequence and step")
    assert a.seqs * a.steps <= kept and 0 <= roots.min() and roots.max() < a.vocab


if __name__ == "__main__":
    main()
