"""The workloads of a hybrid decoder's token mixing: what stands at the place of
the key/value cache's attention in the layers that keep a state of fixed size,
and the positions of the attention layers.

* ``delta``   the gated delta rule (``delta_rule``): for each request and head
              a state S [key_size, value_size] in 32 bits, and token by token
              S <- e^g S, S <- S + k (beta (v - S^T k))^T, o = scale S^T q with
              q and k of length one. A step has one token a request, a few
              (drafted ones), or ragged prompts, and leaves the states updated.
* ``conv``    the short causal convolution over the tokens that such a layer's
              q, k and v go through (``short_conv``), with SiLU and the last
              width - 1 inputs of each request carried from step to step.
* ``rotate``  rotary positions with one or several axes (time, height, width)
              of q and k before they are appended and attended (``rotate_qk``).

With ``own`` false the same is computed in elementary torch operations in 32
bits (angles, and sums of logarithms of decays, in 64). A request without
earlier tokens (``held`` 0) starts from zeros, whatever its state holds.

Head counts are those of the Llama shapes that the benchmark and the tests use
(hidden 4096: 32 heads of 128; hidden 8192: 64 query and 8 key/value heads; a
tensor-parallel shard of them), with as many state heads as there are query
heads, or half of them sharing their keys.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_package = None
CHUNK = 64
EPS = 1e-6  # added to a squared length
MAX_STATE = 64 * 32 * 128 * 128  # state values of the largest decode case
MAX_TOKENS = 8192 * 32  # tokens times heads of the largest prompt


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
        # One token of one conversation (hidden 4096): latency.
        dict(name="delta_decode_b1_h32", op="delta", B=1, tokens=1, fresh=0, heads=16, group=2, dk=128, dv=128, dtype="float16"),
        # A decode batch's states, read and written once.
        dict(name="delta_decode_b61_h32", op="delta", B=61, tokens=61, fresh=3, heads=16, group=2, dk=128, dv=128, dtype="bfloat16"),
        # Four drafted tokens a request to be verified, one tensor-parallel shard, keys of 64.
        dict(name="delta_verify_b96_h4", op="delta", B=96, tokens=384, fresh=0, heads=4, group=1, dk=64, dv=128, dtype="bfloat16"),
        # Ragged prompts and continued ones of a refilled batch, an odd number of tokens.
        dict(name="delta_prompts_b7_3001_h16", op="delta", B=7, tokens=3001, fresh=4, heads=16, group=1, dk=128, dv=128, dtype="float16"),
        # One long prompt (hidden 4096), keys shared by two heads. The largest.
        dict(name="delta_prompt_b1_8192_h32", op="delta", B=1, tokens=8192, fresh=1, heads=16, group=2, dk=128, dv=128, dtype="bfloat16"),
        # One token of each of a decode batch through the convolution: q, k and v side by side.
        dict(name="conv_decode_b64_c8192", op="conv", B=64, tokens=64, fresh=2, channels=8192, width=4, bias=False, dtype="float16"),
        # Ragged prompts, a width and a number of channels that are no powers of two.
        dict(name="conv_prompts_b5_4099_c1544", op="conv", B=5, tokens=4099, fresh=3, channels=1544, width=3, bias=True, dtype="float16"),
        # One long prompt.
        dict(name="conv_prompt_b1_8192_c8192", op="conv", B=1, tokens=8192, fresh=1, channels=8192, width=4, bias=False, dtype="bfloat16"),
        # Text: a token each of a decode batch (hidden 8192).
        dict(name="rotate_decode_b64_h64x8", op="rotate", tokens=64, q_heads=64, kv_heads=8, D=128, R=128, axes=1, adjacent=False, far=131072, dtype="float16"),
        # Half of the dimensions rotate, in adjacent pairs; an odd number of tokens far into a document.
        dict(name="rotate_3001_h32x8_half", op="rotate", tokens=3001, q_heads=32, kv_heads=8, D=128, R=64, axes=1, adjacent=True, far=1000000, dtype="bfloat16"),
        # Images and video: time, height and width (hidden 8192).
        dict(name="rotate_8192_h64x8_3axes", op="rotate", tokens=8192, q_heads=64, kv_heads=8, D=128, R=128, axes=3, adjacent=False, far=20000, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: 1-256 requests, 1-8192 tokens, 1-32 heads of keys and
    values of 64 or 128, 8-8192 channels, up to 64 + 64 rotated heads of 32-256."""
    op = rng.choice(["delta", "delta", "delta", "conv", "rotate"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "rotate":
        while True:
            D = rng.choice([32, 64, 80, 128, 128, 128, 256])
            R = rng.choice([D, D, D // 2])
            kv = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
            q = kv * rng.choice([1, 2, 3, 4, 7, 8])
            tokens = _log_int(rng, 1, 20000)
            if q <= 64 and tokens * (q + kv) * D <= 8192 * 72 * 128:
                return dict(op=op, tokens=tokens, q_heads=q, kv_heads=kv, D=D, R=R, axes=rng.choice([1, 1, 2, 3]),
                            adjacent=rng.random() < 0.3, far=_log_int(rng, 100, 1000000), dtype=dtype)
    kind = rng.random()
    if kind < 0.4:
        B = _log_int(rng, 1, 128)
        tokens = B
    elif kind < 0.55:
        B = _log_int(rng, 1, 128)
        tokens = B * rng.randint(2, 9)
    else:
        tokens = _log_int(rng, 17, 8192)
        B = min(_log_int(rng, 1, 16), tokens)
    fresh = rng.randint(0, B)
    if op == "conv":
        channels = 8 * _log_int(rng, 1, 1024)
        return dict(op=op, B=B, tokens=tokens, fresh=fresh, channels=channels, width=rng.choice([2, 3, 4, 4]),
                    bias=rng.random() < 0.3, dtype=dtype)
    while True:
        heads, group = rng.choice([1, 2, 3, 4, 5, 8, 16, 16, 32]), rng.choice([1, 1, 2, 3, 4])
        dk, dv = rng.choice([64, 128, 128]), rng.choice([64, 128, 128])
        if heads * group <= 32 and B * heads * group * dk * dv <= MAX_STATE and tokens * heads * group <= MAX_TOKENS:
            return dict(op=op, B=B, tokens=tokens, fresh=fresh, heads=heads, group=group, dk=dk, dv=dv, dtype=dtype)


def _shares(total, count):
    """`total` tokens in `count` ragged parts, none empty; equal ones where they are few a request."""
    if total <= 9 * count and total % count == 0:
        return [total // count] * count
    w = [1.0 + (7 * i) % 5 for i in range(count)]
    parts = [1 + int((total - count) * x / sum(w)) for x in w]
    parts[0] += total - sum(parts)
    return parts


def _requests(case, seed):
    """Each request's new tokens and what it held. The seed sets their order
    alone, so that a case's work is the same for every seed."""
    B = case["B"]
    new = _shares(case["tokens"], B)
    held = [0] * case["fresh"] + [100 + 37 * i for i in range(B - case["fresh"])]
    order = np.random.RandomState(seed % 2**31).permutation(B)
    return [new[i] for i in order], [held[i] for i in order]


def _axes(R, axes):
    """Which axis each of the R / 2 frequencies turns by: sections one after another."""
    half = R // 2
    first = half - (axes - 1) * (half // (axes + 1))
    return [0] * first + [a for a in range(1, axes) for _ in range(half // (axes + 1))]


def prepare(case, seed):
    op = case["op"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    if op == "rotate":
        T, D, R, A = case["tokens"], case["D"], case["R"], case["axes"]
        top = torch.tensor([case["far"]] + [200] * (A - 1), device="cuda")  # an image's rows and columns are few
        positions = (torch.rand(A, T, device="cuda", generator=g) * top[:, None]).int()
        rows = rand(T, (case["q_heads"] + 2 * case["kv_heads"]) * D).to(dtype)  # one projection gives q, k and v
        q, k, _ = rows.split([case["q_heads"] * D, case["kv_heads"] * D, case["kv_heads"] * D], 1)
        axis = _axes(R, A)
        frequencies = 10000.0 ** (-2.0 * torch.arange(R // 2, device="cuda") / R)
        return dict(op=op, q=q.unflatten(1, (-1, D)), k=k.unflatten(1, (-1, D)), positions=positions if A > 1 else positions[0],
                    frequencies=frequencies, axis=torch.tensor(axis, dtype=torch.int32, device="cuda") if A > 1 else None,
                    adjacent=case["adjacent"])
    new, held = _requests(case, seed)
    B, T = case["B"], case["tokens"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    single = max(new) == 1
    state = dict(op=op, held=ints(held), offsets=None if single else ints([0] + list(np.cumsum(new))), max_new=max(new))
    if op == "conv":
        C, W = case["channels"], case["width"]
        return dict(state, x=rand(T, C).to(dtype), weight=(0.5 * rand(C, W)).to(dtype), bias=(0.2 * rand(C)).to(dtype) if case["bias"] else None,
                    windows=rand(B, W - 1, C).to(dtype))
    H, G, dk, dv = case["heads"], case["group"], case["dk"], case["dv"]
    rows = rand(T, 2 * H * dk + H * G * dv).to(dtype)  # q, k and v come side by side out of the convolution
    q, k, v = rows.split([H * dk, H * dk, H * G * dv], 1)
    # Heads remember for a few to a few thousand tokens.
    rate = (torch.rand(H * G, device="cuda", generator=g) * 6 - 6).exp()
    return dict(state, q=q.unflatten(1, (H, dk)), k=k.unflatten(1, (H, dk)), v=v.unflatten(1, (H * G, dv)),
                log_decay=-rate * (1 + rand(T, H * G).exp()).log(), beta=rand(T, H * G).sigmoid(), states=0.3 * rand(B, H * G, dk, dv))


def run(state):
    op = state["op"]
    if own:
        dk = _own()
        if op == "rotate":
            rotary = dk.Rotary(state["frequencies"], state["axis"], state["adjacent"])
            return dk.rotate_qk(state["q"], state["k"], state["positions"], rotary)
        if op == "conv":
            y = dk.short_conv(state["x"], state["weight"], state["windows"], state["held"], state["offsets"], state["max_new"], bias=state["bias"])
            return y, state["windows"]
        o = dk.delta_rule(state["q"], state["k"], state["v"], state["log_decay"], state["beta"], state["states"], state["held"],
                          state["offsets"], state["max_new"])
        return o, state["states"]
    if op == "rotate":
        return _rotate(state)
    return _conv(state) if op == "conv" else _delta(state)


def _rotate(state):
    positions, axis = state["positions"], state["axis"]
    turned = positions[:, None] if axis is None else positions[axis.long()].t()
    angle = turned.double() * state["frequencies"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = cos.shape[-1]
    out = []
    for x in (state["q"], state["k"]):
        pairs, rest = x[..., : 2 * half].float(), x[..., 2 * half :]
        a, b = (pairs[..., 0::2], pairs[..., 1::2]) if state["adjacent"] else (pairs[..., :half], pairs[..., half:])
        c, d = a * cos - b * sin, a * sin + b * cos
        y = torch.stack([c, d], -1).flatten(-2) if state["adjacent"] else torch.cat([c, d], -1)
        out.append(torch.cat([y.to(x.dtype), rest], -1))
    return tuple(out)


def _places(state, T):
    """Offsets, new tokens, and of every token its request and its place among the request's new ones."""
    B = state["held"].numel()
    offsets = torch.arange(B + 1, device="cuda") if state["offsets"] is None else state["offsets"].long()
    count = offsets[1:] - offsets[:-1]
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(offsets[1:], t, right=True)
    return offsets, count, b, t - offsets[b]


def _conv(state):
    x, w, windows = state["x"], state["weight"].float(), state["windows"]
    (T, C), W, B = x.shape, w.shape[1], windows.shape[0]
    offsets, count, b, i = _places(state, T)
    old = torch.where((state["held"] > 0)[:, None, None], windows, 0).reshape(B * (W - 1), C)
    every = torch.cat([old, x])  # windows, then tokens
    acc = state["bias"].float() if state["bias"] is not None else 0.0
    for j in range(W):
        at = i - (W - 1) + j  # the token's place in its request, below 0 in the window
        row = torch.where(at < 0, b * (W - 1) + (W - 1) + at, B * (W - 1) + offsets[b] + at)
        acc = acc + every[row].float() * w[:, j]
    s = torch.arange(W - 1, device="cuda")
    at = count[:, None] - (W - 1) + s
    first = torch.arange(B, device="cuda")[:, None] * (W - 1)
    row = torch.where(at < 0, first + (W - 1) + at, B * (W - 1) + offsets[:-1, None] + at)
    windows.copy_(every[row])
    return (acc / (1 + (-acc).exp())).to(x.dtype), windows


def _delta(state):
    v, states = state["v"], state["states"]
    T, (B, Hv, dk, dv), n = v.shape[0], states.shape, state["max_new"]
    G = Hv // state["q"].shape[1]
    offsets, count, b, i = _places(state, T)
    # Requests side by side, padded with tokens that change nothing: [B, Hv, n, ...].
    C = min(n, CHUNK)
    n = -(-n // C) * C
    at = torch.arange(n, device="cuda")
    real = at < count[:, None]
    rows = torch.where(real, offsets[:-1, None] + at, 0)
    side = lambda x: torch.where(real.view(real.shape + (1,) * (x.dim() - 1)), x[rows].float(), 0).transpose(1, 2)  # noqa: E731
    length = lambda x: x * (x.square().sum(-1, keepdim=True) + EPS).rsqrt()  # noqa: E731
    q = (length(side(state["q"])) * dk**-0.5).repeat_interleave(G, 1)
    k = length(side(state["k"])).repeat_interleave(G, 1)
    v, g, beta = side(v), side(state["log_decay"]), side(state["beta"])
    S = torch.where((state["held"] > 0)[:, None, None, None], states, 0)
    if n <= 16:
        out = torch.empty(B, Hv, n, dv, device="cuda")
        for t in range(n):
            S = S * g[:, :, t, None, None].exp()
            u = beta[:, :, t, None] * (v[:, :, t] - (S * k[:, :, t, :, None]).sum(2))
            S = S + k[:, :, t, :, None] * u[:, :, None]
            out[:, :, t] = (S * q[:, :, t, :, None]).sum(2)
    else:
        cut = lambda x: x.unflatten(2, (-1, C))  # noqa: E731
        q, k, v, beta = cut(q), cut(k), cut(v), cut(beta)
        sums = cut(g).double().cumsum(3)
        lower = torch.ones(C, C, dtype=torch.bool, device="cuda").tril()
        decay = torch.where(lower, (sums[..., :, None] - sums[..., None, :]).exp(), 0).float()
        A = torch.where(lower.tril(-1), beta[..., None] * decay * (k @ k.transpose(-1, -2)), 0)
        inverse = torch.eye(C, device="cuda").expand(A.shape).contiguous()
        for r in range(1, C):  # (1 + A)^-1, row after row
            inverse[..., r, :r] = -(A[..., r, None, :r] @ inverse[..., :r, :r])[..., 0, :]
        P = decay * (q @ k.transpose(-1, -2))
        since = sums.exp().float()[..., None]
        until = (sums[..., -1:] - sums).exp().float()[..., None]
        whole = sums[..., -1].exp().float()[..., None, None]
        u, w = inverse @ (beta[..., None] * v), inverse @ (beta[..., None] * since * k)
        out = torch.empty(v.shape, device="cuda")
        for c in range(n // C):
            d = u[:, :, c] - w[:, :, c] @ S
            out[:, :, c] = (q[:, :, c] * since[:, :, c]) @ S + P[:, :, c] @ d
            S = whole[:, :, c] * S + (k[:, :, c] * until[:, :, c]).transpose(-1, -2) @ d
        out = out.flatten(2, 3)
    states.copy_(S)
    return out.transpose(1, 2)[b, i].to(state["v"].dtype), states


def work(case):
    T = case["tokens"]
    if case["op"] == "rotate":
        n = T * (case["q_heads"] + case["kv_heads"])
        return dict(bytes=4.0 * n * case["D"] + 4.0 * case["axes"] * T, flops=3.0 * n * case["R"])
    B, old = case["B"], case["B"] - case["fresh"]
    if case["op"] == "conv":
        C, W = case["channels"], case["width"]
        return dict(bytes=4.0 * T * C + 2.0 * (W - 1) * C * (B + old) + 2.0 * C * W, flops=(2.0 * W + 4) * T * C)
    H, Hv, dk, dv = case["heads"], case["heads"] * case["group"], case["dk"], case["dv"]
    return dict(bytes=4.0 * Hv * dk * dv * (B + old) + T * (4.0 * H * dk + 4.0 * Hv * dv + 8.0 * Hv), flops=7.0 * T * Hv * dk * dv)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotate":
        A, half = case["axes"], case["R"] // 2
        axis = _axes(case["R"], A)
        positions = state["positions"].reshape(A, -1).double()
        turn = torch.stack([positions[axis[i]] * state["frequencies"][i].double() for i in range(half)], 1)
        factor = torch.polar(torch.ones_like(turn), turn)[:, None]
        out = []
        for x in (state["q"].double(), state["k"].double()):
            z = torch.view_as_complex(x[..., : 2 * half].reshape(*x.shape[:2], half, 2)) if case["adjacent"] else torch.complex(x[..., :half].contiguous(), x[..., half : 2 * half].contiguous())
            z = z * factor
            out.append(torch.cat([torch.view_as_real(z).flatten(-2) if case["adjacent"] else torch.cat([z.real, z.imag], -1), x[..., 2 * half :]], -1))
        return tuple(out)
    new, held = _requests(case, seed)
    ends = np.cumsum(new)
    if case["op"] == "conv":
        W, y, kept = case["width"], [], []
        w = state["weight"].double()
        for b, (n, h) in enumerate(zip(new, held)):
            window = state["windows"][b].double() * (h > 0)
            rows = torch.cat([window, state["x"][ends[b] - n : ends[b]].double()])
            z = (rows.unfold(0, W, 1) * w).sum(-1)
            z = z if state["bias"] is None else z + state["bias"].double()
            y.append(z * torch.sigmoid(z))
            kept.append(rows[n:])
        return torch.cat(y), torch.stack(kept)
    # Token by token, all requests side by side.
    Hv, dk, G = case["heads"] * case["group"], case["dk"], case["group"]
    S = state["states"].double()
    S[torch.tensor([h == 0 for h in held], device="cuda")] = 0
    out = torch.empty(state["v"].shape, dtype=torch.float64, device="cuda")
    head = torch.arange(Hv, device="cuda") // G
    unit = lambda x: x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)  # noqa: E731
    q, k, v = unit(state["q"].double()) / math.sqrt(dk), unit(state["k"].double()), state["v"].double()
    alpha, beta = state["log_decay"].double().exp(), state["beta"].double()
    for t in range(max(new)):
        b = [i for i in range(len(new)) if new[i] > t]
        at = torch.tensor([int(ends[i]) - new[i] + t for i in b], device="cuda")
        every = len(b) == len(new)
        part = S if every else S[b]
        kt, qt = k[at][:, head], q[at][:, head]
        part = part * alpha[at][..., None, None]
        u = beta[at][..., None] * (v[at] - torch.einsum("bhk,bhkv->bhv", kt, part))
        part = part + kt[..., None] * u[:, :, None]
        out[at] = torch.einsum("bhk,bhkv->bhv", qt, part)
        if every:
            S = part
        else:
            S[b] = part
    return out, S
