"""append_kv by how many tokens a workgroup looks for runs among (4 to 64, by
tokens times heads), bit for bit: long runs that start in one workgroup, runs
of one wave between them, and tokens without a slot."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle
from test_kv_gpu import DTYPES, _append_case, _back, _cache, _dev, _random_cache

pytestmark = pytest.mark.gpu


def _append_runs(codes, scales, x, slots):
    """kv_oracle.append, a page's heads and tokens at once."""
    page = codes.shape[1]
    live = np.flatnonzero((slots >= 0) & (slots < codes.shape[0] * page))
    order = live[np.argsort(slots[live] // page, kind="stable")]
    for toks in np.split(order, np.flatnonzero(np.diff(slots[order] // page)) + 1):
        p, at = int(slots[toks[0]] // page), slots[toks] % page
        top = np.abs(x[toks]).max((0, 2)) * (np.float32(1.0) / np.float32(127.0))
        old = np.zeros_like(top) if at[0] == 0 else scales[p].copy()
        s = np.maximum(old, top)
        with np.errstate(all="ignore"):
            inv = np.where(s >= np.float32(2.0**-126), np.float32(1.0) / s, np.float32(0.0)).astype(np.float32)
        grew = top > old
        earlier = codes[p, :at[0]].astype(np.float32) * (old * inv)[None, :, None]
        codes[p, :at[0]][:, grew] = np.clip(np.rint(earlier), -127, 127).astype(np.int8)[:, grew]
        codes[p, at] = np.clip(np.rint(x[toks] * inv[None, :, None]), -127, 127).astype(np.int8)
        scales[p] = s


def _spans(page, tokens, seed):
    """Requests of every kind in turn until there are `tokens`: runs longer
    than 8 tokens and within a group of 16, longer ones, whole pages, single
    tokens, starts inside a page."""
    rng = np.random.default_rng(seed)
    kinds = [(0, page), (3, 1), (0, 9), (1, 14), (5, page + 20), (page - 1, 1), (0, 1), (2, 30), (15, 2), (0, 3 * page)]
    spans, n = [], 0
    while n < tokens:
        off, count = kinds[int(rng.integers(len(kinds)))]
        spans.append((off, min(count, tokens - n)))
        n += spans[-1][1]
    return spans


def test_restatement_agrees():
    rng, pages, slots, x = _append_case(1, 16, 3, 64, _spans(16, 300, 1))
    slots[::17] = -1
    before = _random_cache(rng, pages, 16, 3, 64)
    a, b = [t.copy() for t in before], [t.copy() for t in before]
    kv_oracle.append(a[0], a[2], x[0], slots)
    _append_runs(b[0], b[2], x[0], slots)
    for u, w in zip(a, b):
        np.testing.assert_array_equal(u, w)


# heads x tokens for workgroups of 4, 8, 16, 32 and 64 tokens.
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("heads,tokens", [(3, 1500), (24, 400), (32, 600), (32, 1100), (16, 3001), (33, 8200)])
@pytest.mark.parametrize("page,d", [(16, 64), (32, 128), (64, 64), (128, 64)])
def test_append_by_tokens_a_workgroup(page, d, heads, tokens, dtype):
    from decode_kernel import append_kv

    if heads == 33 and d == 128:
        d = 64  # the host's part of it
    rng, pages, slots, x = _append_case(heads + page, page, heads, d, _spans(page, tokens, tokens + page))
    for lo in range(5, tokens - 40, 173):  # single holes, some, and more than a workgroup's share
        slots[lo: lo + (1, 3, 9, 40)[lo % 4]] = -1
    before = _random_cache(rng, pages, page, heads, d)
    xt = [_dev(a, DTYPES[dtype]) for a in x]
    x = [a.float().cpu().numpy() for a in xt]
    cache, want = _cache(*before), [a.copy() for a in before]
    _append_runs(want[0], want[2], x[0], slots)
    _append_runs(want[1], want[3], x[1], slots)
    sd = _dev(slots)
    for _ in range(2):  # a step made twice leaves the same
        append_kv(cache, xt[0], xt[1], sd)
        for g, w in zip(_back(cache), want):
            np.testing.assert_array_equal(g, w)
