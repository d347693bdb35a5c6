"""Gated delta rule and the short convolution before it.

The token mixing of a decoder layer that keeps a state of fixed size for each
request, at the place where a layer with a cache has ``append_kv`` and
``attend_kv``:

    rows = short_conv(w4a16_linear(x, *qkv), taps, windows, held, step.query_offsets, max_query_len)
    q, k, v = rows split into heads
    o = delta_rule(q, k, v, log_decay, beta, states, held, step.query_offsets, max_query_len)

with ``held`` (what each request had before the step) and ``step`` those of
``plan_kv_step``, so that layers of both kinds share one plan. Row b of
``states`` and ``windows`` belongs to place b of the batch; a request that held
nothing starts from zeros, so a place needs no clearing between requests.
Nothing here waits for the GPU or reads from it. The reference has no
counterpart (it holds weights, python/decode_kernel/__init__.py:32-83). Like
``gemv``, the functions run only through the HIP extension
(include/decode_kernel/dk_delta.h), and nothing goes back through them.
"""

from __future__ import annotations

from typing import Optional

import torch

from ._native import ext as _ext

__all__ = ["delta_rule", "short_conv"]


def _most(max_query_len: Optional[int], query_offsets: Optional[torch.Tensor], tokens: int) -> int:
    if max_query_len is not None:
        return max_query_len
    return 1 if query_offsets is None else max(1, tokens)


def delta_rule(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    log_decay: torch.Tensor,
    beta: torch.Tensor,
    states: torch.Tensor,
    held: Optional[torch.Tensor] = None,
    query_offsets: Optional[torch.Tensor] = None,
    max_query_len: Optional[int] = None,
    scale: Optional[float] = None,
    normalize: bool = True,
) -> torch.Tensor:
    """Each request's new tokens through its states, which it updates in place.

    For each request and head, token by token: ``S *= exp(log_decay)``, ``S +=
    outer(k, beta * (v - S.T @ k))``, ``out = scale * S.T @ q``.

    q, k [tokens, qk_heads, key_size] and v [tokens, v_heads, value_size] in
    fp16 or bf16, v_heads a multiple of qk_heads (head h has the keys of head h
    // (v_heads / qk_heads)), sizes of 64 or 128; log_decay (at most 0,
    -inf empties the state) and beta fp32 [tokens, v_heads]; states fp32 [requests, v_heads, key_size, value_size].
    Request b has the rows ``query_offsets[b]:query_offsets[b + 1]`` (offsets
    that decrease anywhere, or leave the rows, give zeros for all and update
    nothing); without query_offsets, one row a request. ``held[b]`` of 0 or less
    starts from a state of zeros (without held, all go on from theirs). A request
    without rows keeps its state; rows of no request (a captured step's places
    past its last token) give 0. ``max_query_len`` (the most rows a request has;
    default: all) picks kernels, the better the closer it is, and changes no result
    beyond rounding.
    ``normalize`` divides q and k by sqrt(|x|^2 + 1e-6). scale: key_size ** -0.5
    by default. States, sums and decays are 32 bits, whichever kernel runs (in a
    prompt's products a state's element has 22 bits, counted from the largest of its
    column). The rule wants beta * |k|^2 of at most 2; beyond, it amplifies what it
    holds, and near 2 with keys that hardly differ nothing fades and 64 tokens of a
    prompt can lose 2e-3 of values and state (150 tokens one by one 1e-4). A NaN
    or infinity stays in its request (one in v in its column); in a prompt it may
    also reach up to 63 tokens before its own.
    """
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _ext().delta_rule(q, k, v, log_decay, beta, states, held, query_offsets,
                             _most(max_query_len, query_offsets, q.shape[0]), scale, normalize)


def short_conv(
    x: torch.Tensor,
    weight: torch.Tensor,
    windows: torch.Tensor,
    held: Optional[torch.Tensor] = None,
    query_offsets: Optional[torch.Tensor] = None,
    max_query_len: Optional[int] = None,
    bias: Optional[torch.Tensor] = None,
    silu: bool = True,
) -> torch.Tensor:
    """The causal convolution of 2, 3 or 4 taps over each request's tokens.

    ``y[t, c] = silu(bias[c] + sum_j weight[c, j] * x[t - (width - 1) + j, c])``
    (``silu=False``: the sum itself). x [tokens, channels] in fp16 or bf16;
    weight [channels, width], bias [channels] and windows [requests, width - 1,
    channels] of the same type. Inputs from before the step come from windows,
    the oldest first, which then hold each request's last ``width - 1`` inputs.
    held, query_offsets and max_query_len as in delta_rule.
    """
    return _ext().short_conv(x, weight, windows, held, query_offsets,
                             _most(max_query_len, query_offsets, x.shape[0]), bias, silu)
