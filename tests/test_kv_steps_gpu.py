"""Whole steps on the paged cache: places without a token, prompts among many
single tokens, and steps that ran out of pages."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv_oracle
from test_kv_gpu import _attend_case, _back, _cache, _check, _dev, _random_cache, _tables

pytestmark = pytest.mark.gpu


# --------------------------------------------------- rows of no sequence
def _run_abi(q, cache, tables, lens, offsets, max_query_len, out):
    """dk_kv_attend on an output of the test's own."""
    from decode_kernel import _abi

    lib = _abi.load()
    t, hq, d = q.shape
    c = _abi.KvCache(k_codes=cache.k_codes.data_ptr(), v_codes=cache.v_codes.data_ptr(), k_scales=cache.k_scales.data_ptr(),
                     v_scales=cache.v_scales.data_ptr(), pages=cache.pages, heads=cache.heads, head_size=d, page_size=cache.page_size)
    b, w = tables.shape
    n = lib.dk_kv_attend_workspace_bytes(t, b, hq, cache.heads, d, w, cache.page_size, max_query_len)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    rc = lib.dk_kv_attend(q.data_ptr(), 0, q.stride(0), q.stride(1), ctypes.byref(c), tables.data_ptr(), w, lens.data_ptr(),
                          offsets.data_ptr(), t, b, hq, max_query_len, 0.125, 1, out.data_ptr(), ws.data_ptr(), n,
                          torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == _abi.DK_OK, lib.dk_last_error().decode()


@pytest.mark.parametrize("tokens,offsets,most", [
    (9, [0, 1, 2, 3], 1), (300, [0, 1, 2, 3], 1), (3, [0, 1, 2, 3], 1), (40, [0, 0, 0, 0], 1), (12, [5, 6, 6, 9], 3),
    (500, [0, 200, 201, 350], 200), (500, [120, 200, 201, 202], 80), (70, [60, 60, 60, 60], 70), (8, [0, 3, 5, 2**30], 3),
    (8, [-4, 3, 5, 7], 3), (10, [2**30] * 4, 1),
])
@pytest.mark.parametrize("d,heads,group", [(64, 2, 2), (128, 1, 5)])
def test_rows_of_no_sequence_are_zero(d, heads, group, tokens, offsets, most):
    # A captured step has a fixed number of places, and fewer tokens in them.
    rng = np.random.default_rng(tokens)
    lens = [100, 60, 400]
    tables, pages = _tables(rng, lens, 16)
    host = _random_cache(rng, pages, 16, heads, d)
    q = _dev(rng.standard_normal((tokens, heads * group, d)).astype(np.float16))
    q[-1, 0, 0] = np.nan  # what stands in such a row is not looked at
    ends = np.clip(offsets, 0, tokens)
    if ends[-1] == tokens:
        q[-1, 0, 0] = 0
    out = torch.full_like(q, np.nan)
    _run_abi(q, _cache(*host), _dev(tables), _dev(np.array(lens, np.int32)), _dev(np.array(offsets, np.int32)), most, out)
    ref, spread = kv_oracle.attend(q.float().cpu().numpy(), *host, tables, lens, ends, 0.125, True)
    nobody = np.isnan(ref).all((1, 2))
    assert nobody.sum() == tokens - (ends[-1] - ends[0])
    assert not out[torch.from_numpy(nobody).cuda()].any()
    live = ~nobody
    _check(out[torch.from_numpy(live).cuda()], ref[live], spread[live], max(lens), 127 * host[3].max(), torch.float16)


def test_no_requests_give_zeros():
    from decode_kernel import KVCache, attend_kv

    q = torch.ones(70, 4, 64, dtype=torch.float16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    for most in (1, 70):
        junk = torch.full((70, 4, 64), float("nan"), dtype=torch.float16, device="cuda")
        del junk  # the output's memory, most likely
        out = attend_kv(q, KVCache.empty(2, 2, 64, 16), none.view(0, 3), none, torch.zeros(1, dtype=torch.int32, device="cuda"), most)
        assert out.shape == q.shape and not out.any()


@pytest.mark.parametrize("requests,tokens,most", [(2, 40, 40), (2, 300, 300), (3, 5, 1), (70, 300, 200), (4096, 4096, 4096), (4096, 4096, 1)])
def test_offsets_that_decrease_give_zeros(requests, tokens, most):
    # Sequences that share rows are more work than the counts hold: none is done.
    rng = np.random.default_rng(requests)
    heads, group, d = 2, 4, 64
    tables = np.zeros((requests, 1024), np.int32)
    host = _random_cache(rng, 3, 16, heads, d)
    offsets = np.zeros(requests + 1, np.int32)
    offsets[1::2] = tokens
    q = _dev(rng.standard_normal((tokens, heads * group, d)).astype(np.float16))
    out = torch.full_like(q, np.nan)
    args = _cache(*host), _dev(tables), torch.full((requests,), 16000, dtype=torch.int32, device="cuda")
    _run_abi(q, *args, _dev(offsets), most, out)
    assert not out.any()
    offsets = np.minimum(np.arange(requests + 1), tokens).astype(np.int32)  # one step back among many
    offsets[-1] = max(int(offsets[-2]) - 1, 0)
    out.fill_(np.nan)
    _run_abi(q, *args, _dev(offsets), most, out)
    assert not out.any()


# --------------------------------------------- prompts among single tokens
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,at", [(65, [0]), (65, [64]), (65, [31, 32, 33]), (130, [0, 2, 129]), (130, [65, 66]),
                                  (257, [0, 4, 5, 128, 256]), (257, [255]), (600, [9, 10, 300])])
def test_prompts_among_single_tokens(b, at, causal):
    # More than 64 requests: a lane adds up several, and the prompts stand at
    # the ends and the middle of what one lane has.
    rng = np.random.default_rng(b + len(at))
    new, lens = [1] * b, [int(x) for x in np.exp(rng.uniform(0, np.log(300), b))]
    for i, p in enumerate(at):
        new[p] = (70, 150, 33, 257, 129)[i]
        lens[p] = new[p] + (0, 200, 1000, 5, 64)[i]
    for p in range(7, b, 19):  # idle places
        if new[p] == 1:
            new[p], lens[p] = 0, 0
    _attend_case(b, lens, new, 1, 4, 64 if causal else 128, 16, "bf16" if b % 2 else "fp16", causal)


def test_prompts_in_every_place():
    # No single tokens at all: every one of 90 requests is attend_many's.
    rng = np.random.default_rng(3)
    new = [int(x) for x in rng.integers(33, 60, 90)]
    _attend_case(4, [n + int(x) for n, x in zip(new, rng.integers(0, 90, 90))], new, 1, 4, 64, 32, "fp16")


@pytest.mark.parametrize("before", [0, 100])
def test_prompt_of_more_than_64_row_tiles(before):
    # 2100 tokens of 8 query heads: 66 row tiles of 256 a head.
    _attend_case(5, [2100 + before, 40], [2100, 1], 1, 8, 64, 64, "fp16")


@pytest.mark.parametrize("group", [1, 2, 3, 5, 6, 7, 12, 16, 20, 33])
def test_prompt_by_group(group):
    # What a row tile's last token sees, for groups that divide its 256 rows and others.
    n = 1400 // group + 129
    _attend_case(group, [n + 333, n], [n, n], 1, group, 64, 16, "bf16")


# ------------------------------------------------------- out of pages
def test_shortage_then_pages_returned():
    # What to do when free_count fell below 0: take back the requests that
    # found no page, set the count to 0, return pages from there.
    from decode_kernel import KVCache, append_kv, attend_kv, plan_kv_step

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    page, heads, d = 16, 1, 64
    cache = KVCache.empty(6, heads, d, page)
    tables = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    free, count, held = torch.arange(6, dtype=torch.int32, device="cuda"), i32(6), i32(0, 0, 0)
    rng = np.random.default_rng(1)
    make = lambda n, h: _dev(rng.standard_normal((n, h, d)).astype(np.float16))  # noqa: E731

    def step(added):
        n = sum(added)
        s = plan_kv_step(tables, held, i32(*added), free, count, page, n)
        q, k, v = make(n, 2), make(n, 1), make(n, 1)
        append_kv(cache, k, v, s.slots)
        o = attend_kv(q, cache, tables, s.seq_lens, s.query_offsets, max(added))
        ref, spread = kv_oracle.attend(q.float().cpu().numpy(), *_back(cache), tables.cpu().numpy(), s.seq_lens.tolist(),
                                       s.query_offsets.tolist(), d**-0.5, True)
        _check(o, ref, spread, 64, 127 * float(cache.v_scales.max()), torch.float16)
        return s

    s = step([32, 16, 40])  # 2 + 1 + 3 pages: all of them
    assert s.free_count.tolist() == [0]
    held, count = s.seq_lens, s.free_count
    s = step([1, 1, 1])  # two pages are missing: requests 0 and 1 find none
    assert s.free_count.tolist() == [-2] and s.slots[:2].tolist() == [-1, -1] and int(s.slots[2]) >= 0
    assert tables[0, 2] == -1 and tables[1, 1] == -1
    # Request 2 ends and its three pages come back; 0 and 1 take their token back.
    back = tables[2, :3].clone()
    tables[2] = -1
    held = torch.stack([s.seq_lens[0] - 1, s.seq_lens[1] - 1, s.seq_lens[2] * 0])
    count = s.free_count.clamp(min=0)
    free[0:3] = back
    count = count + 3
    s = step([1, 1, 9])
    assert s.free_count.tolist() == [0] and (s.slots >= 0).all()
    assert s.seq_lens.tolist() == [33, 17, 9]
    assert sorted([int(tables[0, 2]), int(tables[1, 1]), int(tables[2, 0])]) == sorted(back.tolist())
