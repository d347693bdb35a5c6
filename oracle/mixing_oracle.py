"""Gated delta rule, short convolution and rotary positions in float64, token
by token, from their definitions. Test infrastructure: the tests compare the
kernels against it; the package never imports it."""

from __future__ import annotations

import numpy as np

EPS = 1e-6  # added to a squared length


def _requests(rows, offsets, requests):
    return [(b, b + 1) for b in range(requests)] if offsets is None else list(zip(offsets[:-1], offsets[1:]))


def delta_rule(q, k, v, log_decay, beta, states, held=None, offsets=None, scale=None, normalize=True):
    """Outputs [tokens, v_heads, value_size], the states after the step, and each
    output's reach: scale |q| |its column of the state|, which bounds it."""
    q, k, v, beta = (np.asarray(x, np.float64) for x in (q, k, v, beta))
    decay = np.exp(np.asarray(log_decay, np.float64))
    states = np.array(states, np.float64)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if normalize:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + EPS) for x in (q, k))
    group = states.shape[1] // q.shape[1]
    q, k = np.repeat(q, group, 1), np.repeat(k, group, 1)
    out, reach = np.zeros(v.shape), np.zeros(v.shape)
    for b, (first, last) in enumerate(_requests(len(q), offsets, len(states))):
        if last > first and held is not None and held[b] <= 0:
            states[b] = 0
        s = states[b]
        for t in range(first, last):
            s = s * decay[t][:, None, None]
            u = beta[t][:, None] * (v[t] - np.einsum("hk,hkv->hv", k[t], s))
            s = s + k[t][:, :, None] * u[:, None, :]
            out[t] = scale * np.einsum("hk,hkv->hv", q[t], s)
            reach[t] = scale * np.sqrt((q[t] ** 2).sum(-1, keepdims=True) * (s * s).sum(1))
        states[b] = s
    return out, states, reach


def short_conv(x, weight, windows, held=None, offsets=None, bias=None, silu=True):
    """Outputs [tokens, channels] and the windows after the step."""
    x, weight = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    windows = np.array(windows, np.float64)
    width = weight.shape[1]
    y = np.zeros(x.shape)
    for b, (first, last) in enumerate(_requests(len(x), offsets, len(windows))):
        if last == first:
            continue
        past = np.zeros_like(windows[b]) if held is not None and held[b] <= 0 else windows[b]
        rows = np.concatenate([past, x[first:last]])
        for t in range(first, last):
            z = (rows[t - first : t - first + width] * weight.T).sum(0) + (0 if bias is None else bias)
            y[t] = z / (1 + np.exp(-z)) if silu else z
        windows[b] = rows[len(rows) - (width - 1) :]
    return y, windows


def rotate(x, positions, frequencies, axes=None, adjacent=False, inverse=False):
    """One of q and k [tokens, heads, head_size]; positions [axes, tokens]."""
    x = np.array(x, np.float64)
    positions, frequencies = np.atleast_2d(np.asarray(positions, np.float64)), np.asarray(frequencies, np.float64)
    n = len(frequencies)
    for i in range(n):
        axis = 0 if axes is None else min(max(int(axes[i]), 0), len(positions) - 1)
        angle = positions[axis] * frequencies[i] * (-1 if inverse else 1)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        p, r = (2 * i, 2 * i + 1) if adjacent else (i, n + i)
        a, b = x[..., p].copy(), x[..., r].copy()
        x[..., p], x[..., r] = a * c - b * s, a * s + b * c
    return x
