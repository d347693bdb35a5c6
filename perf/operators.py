"""The workloads the paged 8-bit key/value cache is measured by.

Between the q/k/v projections and the output projection of a decoder layer a
serving program

* ``plan``    gives the step's new tokens their pages and slots, from the
              requests' lengths, once a step (``plan_kv_step``);
* ``append``  writes the step's keys and values into the cache, in 8 bits with
              a scale for each page and head, once a layer (``append_kv``);
* ``attend``  attends over the cache, once a layer (``attend_kv``): one new
              token a sequence, a few, or whole prompts;
* ``read``    takes values out of the cache, to move or export a sequence
              (``read_kv``). Appended pages are read back with it too.

With ``own`` false the same is computed in elementary torch operations in 32
bits. The cache is four tensors: codes int8 k [pages, heads, D/16, page, 16]
and v [pages, heads, D, page], and an fp32 scale for each page and head.

Head counts are those of the Llama shapes that the benchmark and the tests use
(hidden 4096: 32 heads of 128; hidden 8192: 64 query and 8 key/value heads;
one of eight tensor-parallel shards of it: 8 and 1).
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_package = None
QMAX = 127.0
MAX_STORED = 131072 * 8 * 128  # key values the largest decode case reads
MAX_PAIRS = 64 * 4096 * 4096 / 2  # (row, key) pairs of the largest prompt


def _own():
    """This repository's package, imported once."""
    global _package
    if _package is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "decode-kernel_amd"))
        import decode_kernel

        _package = decode_kernel
    return _package


def listed():
    return [
        # One decode step of a full batch: 256 requests, a token each. Latency.
        dict(name="plan_decode_b256", op="plan", B=256, tokens=256, held_lo=1, held_hi=4000, page=16),
        # Prompts of a refilled batch, in one step.
        dict(name="plan_prompts_b37", op="plan", B=37, tokens=30011, held_lo=0, held_hi=900, page=64),
        # One layer's new keys and values of a decode batch; the pages hold tokens already.
        dict(name="append_decode_b200", op="append", B=200, tokens=200, held_lo=1, held_hi=2000, heads=8, D=128, page=16, dtype="float16"),
        # The same of several prompts, ragged, on top of a short shared start.
        dict(name="append_prompts_8003", op="append", B=7, tokens=8003, held_lo=0, held_hi=100, heads=8, D=128, page=64, dtype="bfloat16"),
        # One sequence out of a cache of 32 heads (hidden 4096).
        dict(name="read_5000_h32", op="read", tokens=5000, heads=32, D=128, page=32, dtype="float16"),
        # Many sequences' values, to move them to another card.
        dict(name="read_65000_h8", op="read", tokens=65000, heads=8, D=128, page=16, dtype="bfloat16"),
        # Decode of one short conversation (hidden 4096): the smallest call.
        dict(name="decode_b1_700_h32", op="attend", B=1, new=1, held_lo=700, held_hi=700, idle=0, heads=32, group=1, D=128, page=16, dtype="float16"),
        # Decode of one very long document (hidden 8192).
        dict(name="decode_b1_131071_h8x8", op="attend", B=1, new=1, held_lo=131071, held_hi=131071, idle=0, heads=8, group=8, D=128, page=64, dtype="float16"),
        # A server's decode batch: 61 ragged sequences, three idle places.
        dict(name="decode_b64_ragged_h8x8", op="attend", B=64, new=1, held_lo=33, held_hi=9000, idle=3, heads=8, group=8, D=128, page=16, dtype="float16"),
        # Three drafted tokens a sequence to be verified, one tensor-parallel shard, heads of 64.
        dict(name="verify_b96_h1x8_d64", op="attend", B=96, new=4, held_lo=100, held_hi=12000, idle=0, heads=1, group=8, D=64, page=32, dtype="bfloat16"),
        # A prompt's next pieces on top of long contexts, an odd number of tokens.
        dict(name="chunk_b3_501_h8x4", op="attend", B=3, new=501, held_lo=5000, held_hi=20000, idle=0, heads=8, group=4, D=128, page=32, dtype="bfloat16"),
        # A whole prompt (hidden 8192). The largest.
        dict(name="prompt_b1_4096_h8x8", op="attend", B=1, new=4096, held_lo=4096, held_hi=4096, idle=0, heads=8, group=8, D=128, page=64, dtype="float16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: 1-512 requests, 1-131071 tokens each, one new token a
    sequence, a few, or prompts of up to 4096, pages of 16-128 tokens, 1-32
    key/value heads of 64 or 128, groups of 1-12 query heads."""
    op = rng.choice(["plan", "append", "append", "read", "attend", "attend", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        B = _log_int(rng, 1, 512)
        return dict(op=op, B=B, tokens=B if rng.random() < 0.5 else max(B, _log_int(rng, 1, 30000)), held_lo=rng.choice([0, 1]),
                    held_hi=_log_int(rng, 1, 4000), page=page)
    heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 10, 16, 32])
    D = rng.choice([64, 128, 128])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "append":
        tokens = min(_log_int(rng, 1, 8000), 8003 * 8 * 128 // (heads * D))
        B = min(tokens, _log_int(rng, 1, 256)) if rng.random() < 0.6 else tokens
        return dict(op=op, B=min(B, 256), tokens=min(tokens, 256) if B == tokens else tokens, held_lo=rng.choice([0, 1]),
                    held_hi=_log_int(rng, 1, 500), heads=heads, D=D, page=page, dtype=dtype)
    if op == "read":
        tokens = _log_int(rng, 1, min(65000, 65000 * 8 * 128 // (heads * D)))
        return dict(op=op, tokens=tokens, heads=heads, D=D, page=page, dtype=dtype)
    while True:
        kind = rng.random()
        new = 1 if kind < 0.5 else rng.randint(2, 9) if kind < 0.7 else _log_int(rng, 16, 4096)
        B = _log_int(rng, 1, 256 if new < 16 else 8)
        hi = _log_int(rng, new, 131071 if B == 1 else 20000)
        lo = _log_int(rng, new, hi)
        heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 10, 16, 32])
        group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 8, 12])
        if heads * group <= 64 and B * hi * heads * D <= MAX_STORED and B * new * heads * group * hi <= MAX_PAIRS:
            return dict(op=op, B=B, new=new, held_lo=lo, held_hi=hi, idle=rng.choice([0, 0, B // 8]), heads=heads, group=group,
                        D=D, page=page, dtype=dtype)


def _spread(lo, hi, count):
    """`count` lengths from lo to hi, evenly over their logarithm."""
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * i / max(1, count - 1)))) - 1 for i in range(count)][::-1]


def _shares(total, count):
    """`total` tokens in `count` ragged parts, none empty."""
    w = [1.0 + (7 * i) % 5 for i in range(count)]
    parts = [1 + int((total - count) * x / sum(w)) for x in w]
    parts[0] += total - sum(parts)
    return parts


def _requests(case, seed):
    """Lengths held and new of each request. The seed sets their order alone,
    so that a case's work is the same for every seed."""
    B = case["B"]
    held = _spread(case["held_lo"], case["held_hi"], B)
    new = [case["new"]] * B if "new" in case else _shares(case["tokens"], B)
    for i in range(case.get("idle", 0)):  # places of a batch without a request
        held[i * 7 % B] = 0
    order = np.random.RandomState(seed % 2**31).permutation(B)
    return [held[i] for i in order], [new[i] for i in order]


def _device(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(g, *shape):
    """int8 codes as a page's largest value being 127 leaves them."""
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.float16).mul_(38).round_().clamp_(-127, 127).to(torch.int8)


def _cache(g, pages, case):
    H, D, P = case["heads"], case["D"], case["page"]
    s = lambda mean: mean * (0.3 * torch.randn(pages, H, device="cuda", generator=g)).exp()  # noqa: E731
    return _codes(g, pages, H, D // 16, P, 16), _codes(g, pages, H, D, P), s(1.0 / 38), s(0.5 / 38)


def _tables(g, lens, width, page):
    """Pages in no order, as a server that ran for a while gives them; -1 after
    a request's last page. Returns the tables and how many pages they name."""
    count = _device([-(-n // page) for n in lens], torch.int64)
    taken = sum(-(-n // page) for n in lens)
    ids = torch.randperm(taken + 7, device="cuda", generator=g)[:taken].int()
    col = torch.arange(width, device="cuda")
    tables = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    tables[col < count[:, None]] = ids
    return tables, taken + 7


def _slots(tables, lens_from, lens_to, page):
    """Slots of the tokens lens_from[b] <= t < lens_to[b], request by request."""
    start, count = _device(lens_from, torch.int64), _device([b - a for a, b in zip(lens_from, lens_to)], torch.int64)
    b = torch.repeat_interleave(torch.arange(len(lens_from), device="cuda"), count)
    pos = start[b] + torch.arange(b.numel(), device="cuda") - (count.cumsum(0) - count)[b]
    return tables[b, pos // page].long() * page + pos % page


def prepare(case, seed):
    op, P = case["op"], case["page"]
    g = _generator(seed)
    if op == "read":
        n = case["tokens"]
        tables, pages = _tables(g, [n], -(-n // P), P)
        return dict(op=op, cache=_cache(g, pages, case), slots=_slots(tables, [0], [n], P), dtype=getattr(torch, case["dtype"]))
    held, new = _requests(case, seed)
    if op == "plan":
        lens = [a + b for a, b in zip(held, new)]
        width = -(-max(lens) // P) + 2
        tables, pages = _tables(g, held, width, P)
        need = sum(-(-a // P) - -(-b // P) for a, b in zip(lens, held))
        free = pages + torch.randperm(need + 50, device="cuda", generator=g).int()
        return dict(op=op, tables=tables, held=_device(held), new=_device(new), free=free,
                    free_count=_device([need + 40]), page=P, tokens=case["tokens"])
    dtype = getattr(torch, case["dtype"])
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    if op == "append":
        lens = [a + b for a, b in zip(held, new)]
        start = [a // P * P for a in held]  # pages before a request's last one are not touched
        rel = [a - s for a, s in zip(held, start)]
        end = [n - s for n, s in zip(lens, start)]
        tables, pages = _tables(g, end, -(-max(end) // P), P)
        shape = (case["tokens"], case["heads"], case["D"])
        return dict(op=op, cache=_cache(g, pages, case), slots=_slots(tables, rel, end, P), live=_slots(tables, [0] * len(end), end, P),
                    k=rand(*shape).to(dtype), v=(0.5 * rand(*shape)).to(dtype), dtype=dtype)
    new = [min(n, h) for n, h in zip(new, held)]  # the new tokens are in the cache already
    idle_as_empty = [n if n else (1 if case["new"] == 1 else 0) for n in new]
    width = -(-max(held) // P)
    tables, pages = _tables(g, held, width, P)
    T, Hq = sum(idle_as_empty), case["heads"] * case["group"]
    offsets = None if case["new"] == 1 else _device([0] + list(np.cumsum(idle_as_empty)))
    return dict(op=op, cache=_cache(g, pages, case), tables=tables, lens=_device(held), offsets=offsets, max_new=case["new"],
                q=rand(T, Hq, case["D"]).mul_(1.5).to(dtype))


def run(state):
    op = state["op"]
    if own:
        dk = _own()
        if op == "plan":
            step = dk.plan_kv_step(state["tables"], state["held"], state["new"], state["free"], state["free_count"], state["page"], state["tokens"])
            return state["tables"], step.slots, step.positions, step.query_offsets, step.seq_lens, step.free_count
        cache = dk.KVCache(*state["cache"])
        if op == "append":
            dk.append_kv(cache, state["k"], state["v"], state["slots"])
            return *dk.read_kv(cache, state["live"], dtype=state["dtype"]), cache.k_scales, cache.v_scales
        if op == "read":
            return dk.read_kv(cache, state["slots"], dtype=state["dtype"])
        return dk.attend_kv(state["q"], cache, state["tables"], state["lens"], query_offsets=state["offsets"], max_query_len=state["max_new"])
    if op == "plan":
        return _plan(state)
    if op == "append":
        kc, vc, ks, vs = state["cache"]
        _append(kc, ks, state["k"].float().unflatten(2, (-1, 16)), state["slots"])
        _append(vc, vs, state["v"].float(), state["slots"])
        return *_read(state["cache"], state["live"], state["dtype"]), ks, vs
    if op == "read":
        return _read(state["cache"], state["slots"], state["dtype"])
    return _attend(state)


def _plan(state):
    """New pages come off the end of the free list in the order of the
    requests; a token without a page has slot -1."""
    tables, free, P, n = state["tables"], state["free"], state["page"], state["tokens"]
    width = tables.shape[1]
    held = state["held"].long().clamp(min=0)
    ends = state["new"].long().clamp(min=0).cumsum(0).clamp(max=n)
    offsets = torch.cat([ends.new_zeros(1), ends])
    lens = (held + offsets[1:] - offsets[:-1]).clamp(max=width * P)
    had = (held + P - 1) // P
    need = ((lens + P - 1) // P - had).clamp(min=0)
    rank0 = need.cumsum(0) - need
    token = torch.arange(n, device=tables.device)
    b = torch.searchsorted(ends, token, right=True)
    real = b < held.numel()
    b = b.clamp(max=held.numel() - 1)
    pos = held[b] + token - offsets[b]
    col = pos // P
    inside = real & (col < width)
    rank = rank0[b] + col - had[b]
    count = state["free_count"].long().clamp(max=free.numel())
    fresh = torch.where(rank < count, free[(count - 1 - rank).clamp(0, free.numel() - 1)], -1)
    opens = inside & (pos % P == 0)
    tables[b[opens], col[opens]] = fresh[opens]
    page = tables[b, col.clamp(max=width - 1)].long()
    slots = torch.where(inside & (page >= 0), page * P + pos % P, -1)
    return tables, slots, torch.where(real, pos, -1).int(), offsets.int(), lens.int(), (state["free_count"] - need.sum()).int()


def _append(codes, scales, x, slots):
    """x [tokens, heads, ...] into codes [pages, heads, ..., page, ...]."""
    P = codes.shape[3]
    page, off = slots // P, slots % P
    opens = torch.cat([page.new_ones(1, dtype=torch.bool), page[1:] != page[:-1]])
    part = opens.long().cumsum(0) - 1  # a page's tokens of this step stand together
    pages, first = page[opens], off[opens]
    amax = x.abs().flatten(2).amax(2)
    top = torch.zeros(pages.numel(), x.shape[1], device=x.device).index_reduce_(0, part, amax, "amax")
    before = torch.where(first[:, None] == 0, 0.0, scales[pages])
    scale = torch.maximum(before, top * torch.tensor(1 / QMAX, device=x.device))
    inv = torch.where(scale >= 2.0**-126, 1 / scale, 0.0)
    earlier = torch.arange(P, device=x.device) < first[:, None]
    ratio = (before * inv)[:, :, None, None, None]
    old = codes[pages]  # [runs, heads, a, page(, 16)]
    flat = old if old.dim() == 5 else old.unsqueeze(4)
    kept = torch.where(earlier[:, None, None, :, None], (flat.float() * ratio).round().to(torch.int8), flat)
    codes[pages] = kept.reshape(old.shape)
    q = (x * inv[part].reshape(x.shape[:2] + (1,) * (x.dim() - 2))).round().clamp(-QMAX, QMAX).to(torch.int8)
    codes[page, :, :, off] = q
    scales[pages] = scale


def _read(cache, slots, dtype):
    kc, vc, ks, vs = cache
    page, off = slots // kc.shape[3], slots % kc.shape[3]
    k = kc[page, :, :, off].flatten(2).float() * ks[page][:, :, None]
    v = vc[page, :, :, off].float() * vs[page][:, :, None]
    return k.to(dtype), v.to(dtype)


def _attend(state):
    q, tables, lens = state["q"], state["tables"], state["lens"].long()
    kc, vc, ks, vs = state["cache"]
    (T, Hq, D), (B, W) = q.shape, tables.shape
    H, P, n = kc.shape[1], kc.shape[3], state["max_new"]
    at = tables.clamp(min=0).long()
    k = (kc[at].float() * ks[at][..., None, None, None]).permute(0, 2, 1, 4, 3, 5).reshape(B, H, W * P, D)
    v = (vc[at].float() * vs[at][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, H, W * P, D)
    offsets = state["offsets"]
    offsets = torch.arange(B + 1, device=q.device) if offsets is None else offsets.long()
    count = offsets[1:] - offsets[:-1]
    i = torch.arange(n, device=q.device)
    real = i < count[:, None]
    rows = (offsets[:-1, None] + i).clamp(max=T - 1)
    qb = q[rows].float().reshape(B, n, H, Hq // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D)
    s = (qb * D**-0.5) @ k.transpose(2, 3)
    last = lens[:, None] - count[:, None] + i  # the last key that a row sees
    hidden = torch.arange(W * P, device=q.device) > last[:, :, None]
    s = s.reshape(B, H, Hq // H, n, W * P).masked_fill_(hidden[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(B, H, -1, W * P) @ v).reshape(B, H, Hq // H, n, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)
    out = torch.empty(T, Hq, D, dtype=q.dtype, device=q.device)
    out[rows[real]] = o[real].to(q.dtype)
    return out


def work(case):
    op, P = case["op"], case["page"]
    if op == "read":
        n = case["tokens"] * case["heads"] * case["D"]
        return dict(bytes=2.0 * n + 4.0 * n + 8.0 * case["heads"] * -(-case["tokens"] // P), flops=2 * n)
    held, new = _requests(case, 0)
    if op == "plan":
        fresh = sum(-(-(a + b) // P) - -(-a // P) for a, b in zip(held, new))
        return dict(bytes=12.0 * case["tokens"] + 20.0 * case["B"] + 8.0 * fresh, flops=0)
    if op == "append":
        one = case["heads"] * case["D"]
        live = sum(a % P + b for a, b in zip(held, new))
        touched = sum(-(-(a % P + b) // P) for a, b in zip(held, new))
        return dict(bytes=2.0 * one * (3 * case["tokens"] + 3 * live) + 24.0 * case["heads"] * touched, flops=6.0 * one * case["tokens"] + 2.0 * one * live)
    new = [min(a, b) for a, b in zip(new, held)]
    H, D, Hq = case["heads"], case["D"], case["heads"] * case["group"]
    pairs = sum(b * a - b * (b - 1) // 2 for a, b in zip(held, new))
    pages = sum(-(-a // P) for a in held)
    return dict(bytes=2.0 * H * D * sum(held) + 8.0 * H * pages + 4.0 * pages + 4.0 * Hq * D * sum(new), flops=4.0 * D * Hq * pairs)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None
    kc, vc, ks, vs = state["cache"]
    P, D = case["page"], case["D"]
    if op in ("read", "append"):
        # The whole cache in 64 bits, token by token: [pages * page, heads, D].
        k = kc.double().permute(0, 3, 1, 2, 4).reshape(-1, case["heads"], D)
        v = vc.double().permute(0, 3, 1, 2).reshape(-1, case["heads"], D)
        sk, sv = ks.double(), vs.double()
        if op == "append":
            slots = state["slots"]
            sk, sv = _exact_append(k, sk, state["k"].double(), slots, P), _exact_append(v, sv, state["v"].double(), slots, P)
            slots = state["live"]
        else:
            slots = state["slots"]
        values = k[slots] * sk[slots // P][:, :, None], v[slots] * sv[slots // P][:, :, None]
        return values + (sk, sv) if op == "append" else values
    q, Hq, G = state["q"].double(), case["heads"] * case["group"], case["group"]
    held = state["lens"].tolist()
    offsets = list(range(len(held) + 1)) if state["offsets"] is None else state["offsets"].tolist()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, L in enumerate(held):
        rows = slice(offsets[b], offsets[b + 1])
        n = offsets[b + 1] - offsets[b]
        if L == 0 or n == 0:
            continue
        at = state["tables"][b, : -(-L // P)].long()
        hidden = torch.arange(L, device="cuda") > torch.arange(L - n, L, device="cuda")[:, None]
        for h in range(case["heads"]):
            k = (kc[at, h].double() * ks[at, h].double()[:, None, None, None]).permute(0, 2, 1, 3).reshape(-1, D)[:L]
            v = (vc[at, h].double() * vs[at, h].double()[:, None, None]).transpose(1, 2).reshape(-1, D)[:L]
            for head in range(h * G, h * G + G):
                p = torch.softmax((q[rows, head] @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), dim=1)
                out[rows, head] = p @ v
    return out


def _exact_append(values, scale, x, slots, P):
    """The step in 64 bits: `values` [slots, heads, D] holds codes, `scale` [pages, heads]. Updates the codes; returns the scales."""
    page = slots // P
    grown = scale.clone()
    grown[page[slots % P == 0]] = 0
    before = grown.clone()
    tops = x.abs().amax(2) / 127
    for h in range(x.shape[1]):
        grown[:, h].scatter_reduce_(0, page, tops[:, h], "amax")
    ratio = torch.where(grown > 0, before / grown, 0.0)
    values.copy_((values.view(-1, P, *values.shape[1:]) * ratio[:, None, :, None]).round().view(values.shape))
    values[slots] = (x / grown[page][:, :, None]).round().clamp(-127, 127)
    return grown
