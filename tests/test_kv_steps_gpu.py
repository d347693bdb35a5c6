"""Whole steps on the paged cache: places without a token, prompts among many
single tokens, and steps that ran out of pages."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv_oracle
from test_kv_gpu import _cache, _check, _dev, _random_cache, _tables

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
