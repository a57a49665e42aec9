"""A small decoder whose attention runs on the package's cache operators, driven by the
drop-in generation loops.

    python examples/cached_decoder.py [--tokens 200] [--beams 4]

The decoder is a stand-in with random weights (no positions, no training), in the
reference's decoder protocol (`prefill(embeddings, rows, capacity)` returns a decoding
and the first logits; `step(tokens)`), with three kinds of cache:

  * beams: the prompt's keys and values are computed once and shared by all beams
    (prefix_attention); each beam keeps only its own tokens, and a beam step reorders
    only those (kv_reorder).
  * one long sequence within a budget: each token's attention also accumulates every
    slot's weight (window_attention with `weights`), and when the cache is full the
    lightest slots leave it (kv_evict), so memory and time per token stay bounded.
  * beams over a cache held in 4 bits: every token's keys and values are quantised as they come
    (kv_quantize) and attended as they lie (quantized_attention); a beam step moves the records
    (kv_reorder on the uint8 cache).

The prompt itself runs through window_attention with a sliding window and sinks.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from __graft_entry__ import load_package  # noqa: E402

sv = load_package()


class Weights:
    """Random weights of a decoder with grouped heads."""

    def __init__(self, layers=2, heads=8, kv_heads=2, head_dim=64, vocab=512, dtype=torch.bfloat16, device="cuda",
                 seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.heads, self.kv_heads, self.head_dim, self.vocab = heads, kv_heads, head_dim, vocab
        self.hidden, self.dtype, self.device = heads * head_dim, dtype, device
        width = (heads + 2 * kv_heads) * head_dim

        def make(*shape):
            return (torch.randn(shape, generator=g, device=device) * shape[0] ** -0.5).to(dtype)

        self.layers = [(make(self.hidden, width), make(self.hidden, self.hidden)) for _ in range(layers)]
        self.embedding = torch.randn((vocab, self.hidden), generator=g, device=device).to(dtype)
        self.head = make(self.hidden, vocab)


def forward(w, x, attend):
    """x [rows, n, hidden] through the layers; attend(layer, q, k, v) does the attention,
    q [rows, n, heads, head_dim], k / v [rows, kv_heads, n, head_dim] read in place from
    the fused projection.  Returns the last token's logits [rows, vocab]."""
    H, K, D = w.heads, w.kv_heads, w.head_dim
    for i, (qkv, out) in enumerate(w.layers):
        y = torch.nn.functional.rms_norm(x, (w.hidden,)) @ qkv
        q = y[..., :H * D].unflatten(2, (H, D))
        k = y[..., H * D:(H + K) * D].unflatten(2, (K, D)).transpose(1, 2)
        v = y[..., (H + K) * D:].unflatten(2, (K, D)).transpose(1, 2)
        x = x + attend(i, q, k, v).flatten(2) @ out
    return torch.nn.functional.rms_norm(x[:, -1], (w.hidden,)) @ w.head


class SharedPrefixDecoding:
    """Beams behind one prompt: the prompt's cache is read once for all of them."""

    def __init__(self, w, prefix, rows, capacity):
        self.w, self.prefix, self.length = w, prefix, 0  # prefix: per layer (keys, values) [kv_heads, P, head_dim]
        shape = (len(w.layers), rows, w.kv_heads, max(capacity, 1), w.head_dim)
        self.keys = torch.zeros(shape, dtype=w.dtype, device=w.device)
        self.values = torch.zeros_like(self.keys)

    def step(self, tokens):
        at = self.length
        self.length += 1

        def attend(i, q, k, v):
            self.keys[i, :, :, at:at + 1] = k
            self.values[i, :, :, at:at + 1] = v
            return sv.prefix_attention(q, *self.prefix[i], self.keys[i], self.values[i], self.length)

        return forward(self.w, self.w.embedding[tokens.reshape(-1)][:, None], attend)

    def reorder_device(self, parents):
        sv.kv_reorder(self.keys, self.values, parents, self.length)


class BudgetDecoding:
    """One sequence whose cache holds at most `capacity` slots: when it is full, it is cut
    down to `budget` of them by accumulated attention weight."""

    def __init__(self, w, prompt, capacity, budget, sinks=4, recent=16):
        self.w, self.budget, self.sinks, self.recent = w, budget, sinks, recent
        self.length = self.position = prompt[0][0].shape[1]
        capacity = max(capacity, self.length + 1)
        shape = (len(w.layers), 1, w.kv_heads, capacity, w.head_dim)
        self.keys = torch.zeros(shape, dtype=w.dtype, device=w.device)
        self.values = torch.zeros_like(self.keys)
        for i, (k, v) in enumerate(prompt):
            self.keys[i, 0, :, :self.length], self.values[i, 0, :, :self.length] = k, v
        self.weights = torch.zeros(shape[:-1], dtype=torch.float32, device=w.device)
        self.positions = torch.full(shape[:-1], -1, dtype=torch.int32, device=w.device)
        self.positions[..., :self.length] = torch.arange(self.length, dtype=torch.int32, device=w.device)

    def step(self, tokens):
        if self.length == self.keys.shape[3]:
            cut = sv.kv_evict(self.keys, self.values, self.weights, self.positions, budget=self.budget,
                              sinks=self.sinks, recent=self.recent)
            self.weights, self.positions, self.length = cut["weights"], cut["positions"], self.budget
        at = self.length
        self.length += 1
        self.positions[..., at] = self.position
        self.position += 1

        def attend(i, q, k, v):
            self.keys[i, :, :, at:at + 1] = k
            self.values[i, :, :, at:at + 1] = v
            return sv.window_attention(q, self.keys[i], self.values[i], self.length, weights=self.weights[i])

        return forward(self.w, self.w.embedding[tokens.reshape(-1)][:, None], attend)


class QuantizedDecoding:
    """Beams whose whole cache, the prompt's included, is held in 4 bits."""

    def __init__(self, w, prompt, rows, capacity):
        self.w, self.length = w, prompt[0][0].shape[1]
        shape = (len(w.layers), rows, w.kv_heads, self.length + max(capacity, 1), sv.kv_record_bytes(w.head_dim))
        self.keys = torch.zeros(shape, dtype=torch.uint8, device=w.device)
        self.values = torch.zeros_like(self.keys)
        for i, (k, v) in enumerate(prompt):
            sv.kv_quantize(k.expand(rows, -1, -1, -1), v.expand(rows, -1, -1, -1), self.keys[i], self.values[i],
                           self.length)

    def step(self, tokens):
        self.length += 1

        def attend(i, q, k, v):
            sv.kv_quantize(k, v, self.keys[i], self.values[i], self.length)
            return sv.quantized_attention(q, self.keys[i], self.values[i], self.length)

        return forward(self.w, self.w.embedding[tokens.reshape(-1)][:, None], attend)

    def reorder_device(self, parents):
        sv.kv_reorder(self.keys, self.values, parents, self.length)


class Decoder:
    """The reference's decoder protocol over any of the caches."""

    def __init__(self, w, window=64, sinks=4, budget=None, slack=32, quantized=False):
        self.w, self.window, self.sinks, self.budget, self.slack = w, window, sinks, budget, slack
        self.quantized = quantized

    def prefill(self, embeddings, rows, capacity):
        prompt = []

        def attend(i, q, k, v):
            prompt.append((k[0], v[0]))
            return sv.window_attention(q, k, v, window=self.window, sinks=self.sinks)

        logits = forward(self.w, embeddings, attend)
        new = capacity - embeddings.shape[1]
        if self.quantized:
            return QuantizedDecoding(self.w, prompt, rows, new), logits.expand(rows, -1)
        if self.budget is None:
            return SharedPrefixDecoding(self.w, prompt, rows, new), logits.expand(rows, -1)
        return BudgetDecoding(self.w, prompt, self.budget + self.slack, self.budget), logits


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=200)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=257)
    a = ap.parse_args()
    from starvector_b200 import runtime_shared as rs
    w = Weights()
    g = torch.Generator(device="cuda").manual_seed(1)
    prompt = torch.randn((1, a.prompt, w.hidden), generator=g, device="cuda").to(w.dtype)
    torch.manual_seed(0)
    tokens, why = rs._beam_sample(Decoder(w), prompt, a.tokens, 1.0, 0.9, a.beams, [], None, True, lambda step: None)
    print(f"{a.beams} beams behind a shared prompt of {a.prompt}: {len(tokens)} tokens ({why}), first {tokens[:8]}")
    tokens, why = rs._beam_sample(Decoder(w, quantized=True), prompt, a.tokens, 1.0, 0.9, a.beams, [], None, True,
                                  lambda step: None)
    print(f"{a.beams} beams over a 4-bit cache: {len(tokens)} tokens ({why}), first {tokens[:8]}")
    tokens, why = rs._sample(Decoder(w, budget=128), prompt, a.tokens, 1.0, 0.9, [], None, True, lambda step: None)
    print(f"one sequence within 128 slots: {len(tokens)} tokens ({why}), first {tokens[:8]}")


if __name__ == "__main__":
    main()
