#!/usr/bin/env python3
"""A small hybrid decoder on this package alone: every other layer mixes tokens
by the gated delta rule, the others attend over the paged 8-bit cache.

    PYTHONPATH=decode-kernel_amd python examples/hybrid_decode.py [--layers 4] [--tokens 24]

Random weights, a batch of ragged prompts and one idle place. One plan_kv_step a
step serves all layers: its offsets and what the requests held before say which
rows belong to whose state, its slots and lengths which keys are whose. A delta
layer is w4a16_linear (q, k, v side by side), short_conv, delta_rule and
w4a16_linear; an attention layer w4a16_linear, rotate_qk, append_kv, attend_kv
and w4a16_linear; both end in the fused MLP. --check runs the sequences again in
one step and compares the last tokens' logits.
"""

from __future__ import annotations

import argparse

import torch
import torch.nn.functional as F

from decode_kernel import (KVCache, QuantizedMLP, Rotary, append_kv, attend_kv, delta_rule, plan_kv_step,
                           quantize_and_pack, rotate_qk, short_conv, w4a16_linear)


class Hybrid:
    def __init__(self, layers=4, hidden=512, heads=8, kv_heads=2, head_size=64, inner=1024, vocab=1000, width=4, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
        w = lambda m, k: rand(m, k) * k**-0.5  # noqa: E731
        self.heads, self.kv_heads, self.head_size = heads, kv_heads, head_size
        self.key_heads = heads // 2  # two heads of a state share their keys
        self.channels = (2 * self.key_heads + heads) * head_size
        self.embed = rand(vocab, hidden).half()
        self.layers = []
        for i in range(layers):
            delta = i % 2 == 0
            rows = self.channels if delta else (heads + 2 * kv_heads) * head_size
            self.layers.append(dict(
                delta=delta, qkv=quantize_and_pack(w(rows, hidden)), out=quantize_and_pack(w(hidden, heads * head_size)),
                mlp=QuantizedMLP.from_float(w(inner, hidden), w(inner, hidden), w(hidden, inner)),
                gates=w(2 * heads, hidden).half(), rate=torch.linspace(-4, 0, heads, device="cuda").exp(),
                taps=(0.5 * rand(self.channels, width)).half() if delta else None))
        self.width = width
        self.head = quantize_and_pack(w(vocab, hidden))
        self.rotary = Rotary.from_base(head_size)

    def _norm(self, x):
        return (x.float() * x.float().square().mean(-1, keepdim=True).add(1e-6).rsqrt()).half()

    def _delta(self, x, layer, memory, held, step, most):
        d = self.head_size
        rows = short_conv(w4a16_linear(x, *layer["qkv"]), layer["taps"], memory["windows"], held, step.query_offsets, most)
        q, k, v = (t.unflatten(1, (-1, d)) for t in rows.split([self.key_heads * d, self.key_heads * d, self.heads * d], 1))
        a, b = (x @ layer["gates"].t()).float().chunk(2, 1)
        return delta_rule(q, k, v, -layer["rate"] * F.softplus(a), b.sigmoid(), memory["states"], held, step.query_offsets, most)

    def _attend(self, x, layer, cache, tables, step, most):
        d = self.head_size
        rows = w4a16_linear(x, *layer["qkv"])
        q, k, v = (t.unflatten(1, (-1, d)) for t in rows.split([self.heads * d, self.kv_heads * d, self.kv_heads * d], 1))
        q, k = rotate_qk(q, k, step.positions, self.rotary)
        append_kv(cache, k, v, step.slots)
        return attend_kv(q, cache, tables, step.seq_lens, step.query_offsets, most)

    def step(self, tokens, batch, held, step, most):
        """Logits of every token of a planned step; held is what the places had before it."""
        x = self.embed[tokens]
        for layer, memory in zip(self.layers, batch.memory):
            y = self._norm(x)
            o = self._delta(y, layer, memory, held, step, most) if layer["delta"] else self._attend(y, layer, memory, batch.tables, step, most)
            x = x + w4a16_linear(o.flatten(1), *layer["out"])
            x = x + layer["mlp"](self._norm(x))
        return w4a16_linear(self._norm(x), *self.head)


class Batch:
    """What a batch's places keep: pages and tables for the attention layers, a
    state and a window for each delta layer. Neither states nor windows are
    cleared between requests: one that held nothing starts from zeros."""

    def __init__(self, model, places, longest, page_size=16):
        width = -(-longest // page_size)
        self.page_size = page_size
        self.memory = [
            dict(states=torch.randn(places, model.heads, model.head_size, model.head_size, device="cuda"),
                 windows=torch.randn(places, model.width - 1, model.channels, device="cuda").half()) if layer["delta"]
            else KVCache.empty(places * width, model.kv_heads, model.head_size, page_size) for layer in model.layers]
        self.tables = torch.full((places, width), -1, dtype=torch.int32, device="cuda")
        self.held = torch.zeros(places, dtype=torch.int32, device="cuda")
        self.free = torch.arange(places * width, dtype=torch.int32, device="cuda")
        self.free_count = torch.tensor([places * width], dtype=torch.int32, device="cuda")

    def run(self, model, tokens, added, most):
        step = plan_kv_step(self.tables, self.held, added, self.free, self.free_count, self.page_size, tokens.numel())
        logits = model.step(tokens, self, self.held, step, most)
        self.held, self.free_count = step.seq_lens, step.free_count
        return logits, step


def run_prompts(model, batch, prompts):
    """The prompts in one step; each place's last logits (an idle one's are any row's)."""
    counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    ids = torch.tensor([t for p in prompts for t in p], device="cuda")
    logits, step = batch.run(model, ids, counts, max(map(len, prompts)))
    return logits[(step.query_offsets[1:].long() - 1).clamp(min=0)]


def generate(model, prompts, tokens):
    """Greedy continuations [places, tokens] of the prompts (lists of ids, an
    empty one for an idle place), the last step's logits and the batch."""
    batch = Batch(model, len(prompts), max(map(len, prompts)) + tokens)
    last = run_prompts(model, batch, prompts)
    live = torch.tensor([int(len(p) > 0) for p in prompts], dtype=torch.int32, device="cuda")
    rows = torch.tensor([i for i, p in enumerate(prompts) if p], device="cuda")
    row_of = (live.cumsum(0) - 1).clamp(min=0)
    out = []
    for _ in range(tokens):
        ids = last.argmax(-1)
        out.append(ids)
        logits, _ = batch.run(model, ids[rows], live, 1)
        last = logits[row_of]
    if int(batch.free_count) < 0:  # the one look that the host takes
        raise RuntimeError(f"{-int(batch.free_count)} pages were missing")
    return torch.stack(out, 1), last, batch


def again(model, prompts, out):
    """The last tokens' logits from one step over prompts and continuations, and the batch."""
    whole = [p + o if p else [] for p, o in zip(prompts, out.tolist())]
    batch = Batch(model, len(whole), max(map(len, whole)))
    return run_prompts(model, batch, whole), batch


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--check", action="store_true", help="run the sequences again in one step")
    args = ap.parse_args()
    model = Hybrid(args.layers)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1000, (n,), generator=g).tolist() for n in (37, 5, 0, 130, 64)]
    out, last, _ = generate(model, prompts, args.tokens)
    for prompt, ids in zip(prompts, out.tolist()):
        print(f"prompt of {len(prompt)}:", "idle" if not prompt else " ".join(map(str, ids[:12])), "..." * bool(prompt))
    if args.check:
        live = [i for i, p in enumerate(prompts) if p]
        want = again(model, prompts, out)[0][live].float()
        print(f"logits against one step over the whole sequences: {((last[live].float() - want).norm() / want.norm()).item():.1e} apart")


if __name__ == "__main__":
    main()
