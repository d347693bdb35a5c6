"""Attention calls near the largest that are taken: long prompts, wide tables."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,width", [([131072], 2048), ([16384] * 8, 2048), ([9000, 1, 1, 70000, 300], 2048)])
def test_long_prompts(lens, width):
    # 64 query and 8 key/value heads; tables of 131072 keys. The keys of all
    # sequences come from the same pages, in another order each.
    from decode_kernel import KVCache, attend_kv

    page, heads, group, d = 64, 8, 8, 64
    g = torch.Generator(device="cuda").manual_seed(len(lens))
    pages = max(lens) // page + 1
    code = lambda *s: torch.randint(-127, 128, s, device="cuda", generator=g, dtype=torch.int8)  # noqa: E731
    scale = lambda: (0.2 * torch.randn(pages, heads, device="cuda", generator=g)).exp() / 73  # noqa: E731
    cache = KVCache(code(pages, heads, d // 16, page, 16), code(pages, heads, d, page), scale(), scale())
    tables = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        tables[b, : -(-n // page)] = torch.randperm(pages, device="cuda", generator=g)[: -(-n // page)].int()
    offsets = np.concatenate([[0], np.cumsum(lens)])
    q = torch.randn(sum(lens), heads * group, d, device="cuda", generator=g, dtype=torch.float16)
    got = attend_kv(q, cache, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                    torch.tensor(offsets, dtype=torch.int32, device="cuda"), max(lens))
    for b, n in enumerate(lens):
        at = tables[b, : -(-n // page)].long()
        rows = torch.tensor(sorted({0, min(1, n - 1), n // 3, min(16383, n - 1), n - 1}), device="cuda")
        hidden = torch.arange(n, device="cuda") > rows[:, None]
        for h in (0, heads - 1):
            k = (cache.k_codes[at, h].double() * cache.k_scales[at, h].double()[:, None, None, None]).permute(0, 2, 1, 3).reshape(-1, d)[:n]
            v = (cache.v_codes[at, h].double() * cache.v_scales[at, h].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:n]
            for j in (0, group - 1):
                x = q[offsets[b] + rows, h * group + j].double()
                p = ((x @ k.T) * d**-0.5).masked_fill(hidden, -torch.inf).softmax(1)
                ref, spread = p @ v, p @ v.abs()
                # Half a step of fp16, and 2^-14 for the fp32 of scores and sums
                # over up to 2048 tiles; no weight is under 2^-24 of a row's largest.
                half = 0.5 * torch.exp2((ref.abs().clamp(min=1e-30).log2().floor() - 10).clamp(min=-24))
                err = (got[offsets[b] + rows, h * group + j].double() - ref).abs()
                assert (err <= half + 2.0**-14 * spread).all(), (b, h, j, (err / (half + 2.0**-14 * spread)).max().item())


def test_too_large_is_refused():
    from decode_kernel import KVCache, attend_kv

    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros(2**17, 64, 64, dtype=torch.float16, device="cuda")
    tables = torch.zeros(1, 2**15, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="too large"):  # 16 times what the first prompt above has
        attend_kv(q.view(2**21, 4, 64), KVCache.empty(1, 4, 64, 64), tables, i32(64), i32(0, 2**21), 2**21)
