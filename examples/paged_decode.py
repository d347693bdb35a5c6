#!/usr/bin/env python3
"""A small decoder on this package alone: 4-bit projections and MLP, and
between them the paged 8-bit key/value cache.

    PYTHONPATH=decode-kernel_amd python examples/paged_decode.py [--layers 2] [--tokens 24]

Random weights, a batch of ragged prompts and one idle place. The prompts go
through in one step, then every sequence gets a token a step. A step is one
plan_kv_step, whose slots, offsets and lengths all layers share, and for each
layer w4a16_linear (q, k and v at once), append_kv, attend_kv, w4a16_linear
and the fused MLP. Lengths, tables and the free list stay on the GPU; the host
looks at them once, at the end, to see that no page was missing. --check runs
the sequences again in one step and compares the last tokens' logits.
"""

from __future__ import annotations

import argparse

import torch

from decode_kernel import (KVCache, QuantizedMLP, append_kv, attend_kv, plan_kv_step, quantize_and_pack,
                           w4a16_linear)


class Decoder:
    def __init__(self, layers=2, hidden=512, q_heads=8, kv_heads=2, head_size=64, inner=1024, vocab=1000, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        w = lambda m, k: torch.randn(m, k, device="cuda", generator=g) * k**-0.5  # noqa: E731
        self.q_heads, self.kv_heads, self.head_size = q_heads, kv_heads, head_size
        self.embed = torch.randn(vocab, hidden, device="cuda", generator=g).half()
        self.layers = [
            (quantize_and_pack(w((q_heads + 2 * kv_heads) * head_size, hidden)),
             quantize_and_pack(w(hidden, q_heads * head_size)),
             QuantizedMLP.from_float(w(inner, hidden), w(inner, hidden), w(hidden, inner)))
            for _ in range(layers)]
        self.head = quantize_and_pack(w(vocab, hidden))
        self.freqs = 10000.0 ** (-torch.arange(0, head_size, 2, device="cuda") / head_size)

    def _norm(self, x):
        return (x.float() * x.float().square().mean(-1, keepdim=True).add(1e-6).rsqrt()).half()

    def _rotate(self, x, positions):
        angle = positions[:, None, None].float() * self.freqs
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()], -1).half()

    def step(self, tokens, step, caches, tables, max_query_len):
        """Logits of every token of a planned step."""
        x = self.embed[tokens]
        q_size, kv_size = self.q_heads * self.head_size, self.kv_heads * self.head_size
        positions = step.positions.clamp(min=0)
        for (qkv, out, mlp), cache in zip(self.layers, caches):
            rows = w4a16_linear(self._norm(x), *qkv)
            q, k, v = (t.unflatten(1, (-1, self.head_size)) for t in rows.split([q_size, kv_size, kv_size], 1))
            append_kv(cache, self._rotate(k, positions), v, step.slots)
            o = attend_kv(self._rotate(q, positions), cache, tables, step.seq_lens, step.query_offsets, max_query_len)
            x = x + w4a16_linear(o.flatten(1), *out)
            x = x + mlp(self._norm(x))
        return w4a16_linear(self._norm(x), *self.head)


class Batch:
    """A batch's pages: the tables, the free list and what each place holds."""

    def __init__(self, model, places, pages, page_size, width):
        self.caches = [KVCache.empty(pages, model.kv_heads, model.head_size, page_size) for _ in model.layers]
        self.tables = torch.full((places, width), -1, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(places, dtype=torch.int32, device="cuda")
        self.free = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.free_count = torch.tensor([pages], dtype=torch.int32, device="cuda")

    def plan(self, added, num_tokens):
        step = plan_kv_step(self.tables, self.held, added, self.free, self.free_count,
                            self.caches[0].page_size, num_tokens)
        self.held, self.free_count = step.seq_lens, step.free_count
        return step


def generate(model, prompts, tokens, page_size=16):
    """Greedy continuations [places, tokens] of the prompts (lists of ids, an
    empty one for an idle place) and the last step's logits."""
    places = len(prompts)
    longest = max(map(len, prompts)) + tokens
    width = -(-longest // page_size)
    batch = Batch(model, places, places * width, page_size, width)
    counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    ids = torch.tensor([t for p in prompts for t in p], device="cuda")
    step = batch.plan(counts, ids.numel())
    logits = model.step(ids, step, batch.caches, batch.tables, max(map(len, prompts)))
    # Each place's last token; an idle place takes any row, and stays idle.
    last = logits[(step.query_offsets[1:].long() - 1).clamp(min=0)]
    live = (counts > 0).int()
    slot_of = (live.cumsum(0) - live).long()  # the place's row in a decode step
    number = int(sum(len(p) > 0 for p in prompts))
    out = []
    for _ in range(tokens):
        ids = last.argmax(-1)
        out.append(ids)
        step = batch.plan(live, number)
        rows = torch.zeros(number, dtype=ids.dtype, device="cuda").index_add_(
            0, slot_of.clamp(max=number - 1), ids * live)
        last = model.step(rows, step, batch.caches, batch.tables, 1)[slot_of.clamp(max=number - 1)]
    if int(batch.free_count) < 0:  # the one look that the host takes
        raise RuntimeError(f"{-int(batch.free_count)} pages were missing")
    return torch.stack(out, 1), last


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--check", action="store_true", help="run the sequences again in one step")
    args = ap.parse_args()
    model = Decoder(args.layers)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (37, 5, 0, 130, 64)]
    out, last = generate(model, prompts, args.tokens)
    for prompt, ids in zip(prompts, out.tolist()):
        print(f"prompt of {len(prompt)}:", "idle" if not prompt else " ".join(map(str, ids[:12])), "..." * bool(prompt))
    if args.check:
        again, _ = last_logits(model, prompts, out)
        live = [i for i, p in enumerate(prompts) if p]
        err = (again[live] - last[live]).float().norm() / last[live].float().norm()
        print(f"logits against one step over the whole sequences: {err.item():.1e} apart")


def last_logits(model, prompts, out, page_size=16):
    """The last tokens' logits from one step over prompts and continuations."""
    whole = [p + o if p else [] for p, o in zip(prompts, out.tolist())]
    width = -(-max(map(len, whole)) // page_size)
    batch = Batch(model, len(whole), len(whole) * width, page_size, width)
    counts = torch.tensor([len(p) for p in whole], dtype=torch.int32, device="cuda")
    ids = torch.tensor([t for p in whole for t in p], device="cuda")
    step = batch.plan(counts, ids.numel())
    logits = model.step(ids, step, batch.caches, batch.tables, max(map(len, whole)))
    return logits[(step.query_offsets[1:].long() - 1).clamp(min=0)], batch


if __name__ == "__main__":
    main()
