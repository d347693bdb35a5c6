"""numpy restatement of the paged 8-bit key/value cache and its attention.

TEST INFRASTRUCTURE ONLY. Written token by token and page by page from the
definitions in include/decode_kernel/dk_kv.h, without the package's code. The
cache is held here in its plain order, values [pages, page_size, heads,
head_size] int8 and scales [pages, heads]; `to_device_layout` gives the
layouts of the header.
"""

from __future__ import annotations

import numpy as np


def to_device_layout(k: np.ndarray, v: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """[pages, page_size, heads, D] codes -> the header's k_codes and v_codes."""
    n, p, h, d = k.shape
    kc = k.reshape(n, p, h, d // 16, 16).transpose(0, 2, 3, 1, 4)
    return np.ascontiguousarray(kc), np.ascontiguousarray(v.transpose(0, 2, 3, 1))


def from_device_layout(kc: np.ndarray, vc: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    n, h, c, p, _ = kc.shape
    k = kc.transpose(0, 3, 1, 2, 4).reshape(n, p, h, c * 16)
    return np.ascontiguousarray(k), np.ascontiguousarray(vc.transpose(0, 3, 1, 2))


def plan(tables, held, added, free_pages, free_count, page, tokens):
    """One request and one token after the other. Returns (tables, slots,
    positions, query_offsets, seq_lens, free_count)."""
    tables = tables.copy()
    width = tables.shape[1]
    slots = np.full(tokens, -1, np.int64)
    positions = np.full(tokens, -1, np.int32)
    offsets, lens = [0], []
    left = int(free_count)
    for b in range(len(held)):
        had = max(int(held[b]), 0)
        n = min(max(int(added[b]), 0), tokens - offsets[-1])
        for i in range(n):
            t, pos = offsets[-1] + i, had + i
            positions[t] = pos
            col = pos // page
            if col >= width:
                continue
            if col >= -(-had // page) and pos % page == 0:
                left -= 1
                top = left if free_count <= len(free_pages) else left - (free_count - len(free_pages))
                tables[b, col] = free_pages[top] if top >= 0 else -1
            if tables[b, col] >= 0:
                slots[t] = int(tables[b, col]) * page + pos % page
        offsets.append(offsets[-1] + n)
        lens.append(min(had + n, width * page))
    return tables, slots, positions, np.array(offsets, np.int32), np.array(lens, np.int32), left


def append(codes, scales, x, slots):
    """x [tokens, heads, D] float32 into codes [pages, page, heads, D] and
    scales [pages, heads], in place, in fp32 arithmetic: bit for bit."""
    page = codes.shape[1]
    runs = {}  # page -> the step's tokens on it
    for t, s in enumerate(slots):
        if 0 <= s < codes.shape[0] * page:
            runs.setdefault(int(s // page), []).append(t)
    for p, toks in runs.items():
        off = int(slots[toks[0]] % page)
        for h in range(codes.shape[2]):
            new = x[toks, h].astype(np.float32)
            with np.errstate(all="ignore"):
                top = np.float32(np.abs(new).max()) * (np.float32(1.0) / np.float32(127.0))
                if not np.isfinite(top):
                    top = np.float32(np.nan)
                old = np.float32(0.0) if off == 0 else np.float32(scales[p, h])
                s = np.maximum(old, top)  # propagates NaN
                inv = np.float32(1.0) / s if s >= np.float32(2.0**-126) else np.float32(0.0)
                if top > old or np.isnan(top) and not np.isnan(old):
                    ratio = old * inv
                    codes[p, :off, h] = _code(codes[p, :off, h].astype(np.float32) * ratio)
                scales[p, h] = s
                for t in toks:
                    codes[p, int(slots[t] % page), h] = _code(x[t, h].astype(np.float32) * inv)


def _code(y: np.ndarray) -> np.ndarray:
    y = np.where(np.isnan(y), -127.0, y)
    return np.clip(np.rint(y), -127, 127).astype(np.int8)


def read(codes, scales, slots):
    """[tokens, heads, D] = code * scale in float64; zeros outside the cache."""
    page = codes.shape[1]
    out = np.zeros((len(slots), codes.shape[2], codes.shape[3]))
    for t, s in enumerate(slots):
        if 0 <= s < codes.shape[0] * page:
            out[t] = codes[s // page, s % page].astype(np.float64) * scales[s // page][:, None].astype(np.float64)
    return out


def attend(q, k_codes, v_codes, k_scales, v_scales, tables, lens, offsets, scale, causal):
    """q [tokens, q_heads, D] -> (out, spread) in float64. spread is the
    weighted mean of |v|, which the error of rounded weights goes by; rows of
    no sequence are NaN."""
    page, heads, d = k_codes.shape[1:]
    group = q.shape[1] // heads
    out = np.full(q.shape, np.nan)
    spread = np.full(q.shape, np.nan)
    for b, length in enumerate(lens):
        length = min(max(int(length), 0), tables.shape[1] * page)
        n = offsets[b + 1] - offsets[b]
        pages = tables[b, np.arange(length) // page] if length else np.zeros(0, int)
        seen = (pages >= 0) & (pages < k_codes.shape[0])
        at = np.where(seen, pages, 0)
        inside = np.arange(length) % page
        for h in range(heads):
            k = k_codes[at, inside, h].astype(np.float64) * k_scales[at, h][:, None]
            v = v_codes[at, inside, h].astype(np.float64) * v_scales[at, h][:, None]
            for i in range(n):
                keys = seen & (np.arange(length) < (length - n + i + 1 if causal else length))
                rows = slice(h * group, (h + 1) * group)
                if not keys.any():
                    out[offsets[b] + i, rows] = spread[offsets[b] + i, rows] = 0
                    continue
                qi = q[offsets[b] + i, rows].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = scale * (qi @ k[keys].T)
                    p = np.exp(s - s.max(1, keepdims=True))
                    p /= p.sum(1, keepdims=True)
                    out[offsets[b] + i, rows] = p @ v[keys]
                    spread[offsets[b] + i, rows] = p @ np.abs(v[keys])
    return out, spread
