"""Paged key/value cache in 8 bits and the attention over it.

A decoder layer's step between its q/k/v projections and its output
projection (both ``w4a16_linear``):

    step = plan_kv_step(tables, held, added, free_pages, free_count, cache.page_size, tokens)
    append_kv(cache, k, v, step.slots)             # once a layer
    o = attend_kv(q, cache, tables, step.seq_lens, step.query_offsets, max_query_len)

The cache is int8 codes with one fp32 scale for each page (page_size tokens of
one sequence) and head, keys and values apart. A sequence's pages are named by
its row of a block table, -1 for none; token t is at slot
``table[t // page_size] * page_size + t % page_size``. Nothing here waits for
the GPU or reads from it: lengths, tables and the free list stay on the
device, so a step can be captured in a graph. The reference has no counterpart
(it holds weights, python/decode_kernel/__init__.py:32-83). Like ``gemv``, the
functions run only through the HIP extension (include/decode_kernel/dk_kv.h).
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch

from ._native import ext as _ext

__all__ = ["KVCache", "KVStep", "append_kv", "attend_kv", "plan_kv_step", "read_kv"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


@dataclass
class KVCache:
    """One layer's cache. The codes' layout is the one the attention kernels
    read matrix operands in."""

    k_codes: torch.Tensor   # int8 [pages, heads, head_size / 16, page_size, 16]
    v_codes: torch.Tensor   # int8 [pages, heads, head_size, page_size]
    k_scales: torch.Tensor  # fp32 [pages, heads]
    v_scales: torch.Tensor  # fp32 [pages, heads]

    @classmethod
    def empty(cls, pages: int, heads: int, head_size: int = 128, page_size: int = 64,
              device: torch.device | str = "cuda") -> "KVCache":
        """A cache of zeros. head_size 64 or 128; page_size 16, 32, 64 or 128."""
        if head_size not in (64, 128):
            raise ValueError(f"head_size={head_size} must be 64 or 128")
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size={page_size} must be 16, 32, 64 or 128")
        return cls(
            torch.zeros(pages, heads, head_size // 16, page_size, 16, dtype=torch.int8, device=device),
            torch.zeros(pages, heads, head_size, page_size, dtype=torch.int8, device=device),
            torch.zeros(pages, heads, device=device),
            torch.zeros(pages, heads, device=device),
        )

    @property
    def pages(self) -> int:
        return int(self.k_codes.shape[0])

    @property
    def heads(self) -> int:
        return int(self.k_codes.shape[1])

    @property
    def head_size(self) -> int:
        return int(self.v_codes.shape[2])

    @property
    def page_size(self) -> int:
        return int(self.k_codes.shape[3])


class KVStep(NamedTuple):
    """What plan_kv_step gives, all on the device."""

    slots: torch.Tensor          # int64 [num_tokens], -1 for a token without a place
    positions: torch.Tensor      # int32 [num_tokens], its place in its sequence
    query_offsets: torch.Tensor  # int32 [requests + 1], where each request's tokens start
    seq_lens: torch.Tensor       # int32 [requests], tokens held after the step
    free_count: torch.Tensor     # int32 [1], pages left; negative by what was missing


def plan_kv_step(
    block_tables: torch.Tensor,
    held: torch.Tensor,
    added: torch.Tensor,
    free_pages: torch.Tensor,
    free_count: torch.Tensor,
    page_size: int,
    num_tokens: int,
) -> KVStep:
    """Gives the step's new tokens their pages and slots.

    Request b holds ``held[b]`` tokens and gets ``added[b]`` (int32, on the
    device), request after request, ``num_tokens`` places in all: tokens past
    that are left out, places past the last token have slot -1. New pages come
    off the end of ``free_pages[:free_count]`` and are written into
    ``block_tables`` (int32 [requests, width], in place). Check that
    ``free_count`` did not become negative before trusting the step's last
    tokens: those without a page are neither stored nor attended to, and a -1 in
    the tables is not filled in later. Then take those tokens off the next step's
    ``held`` (or drop their requests), and go on from a count of 0: pages are put
    back at ``free_pages[0]``, not below it. The five results share one allocation:
    clone ``seq_lens`` or ``free_count`` to keep them without the slots. At most
    4096 requests.
    """
    return KVStep(*_ext().plan_kv_step(block_tables, held, added, free_pages, free_count,
                                       int(page_size), int(num_tokens)))


def append_kv(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes k and v [tokens, heads, head_size] (fp16 or bf16) at ``slots``.

    A page's scale for a head is the largest ``amax * (1 / 127)`` it has seen
    since its first token was written, a code ``rint(x * (1 / scale))``; where it grows, the page's earlier codes are
    rounded again to the new scale. Tokens of one page stand together and in
    order in ``slots``, as plan_kv_step gives them; slots of -1 are skipped.
    """
    _ext().append_kv(cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, k, v, slots)


def read_kv(cache: KVCache, slots: torch.Tensor,
            dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """k and v [tokens, heads, head_size] at ``slots`` in fp16, bf16 or fp32;
    zeros at a slot of -1. For moving, exporting or checking sequences; the
    attention kernels never do this."""
    if dtype not in _DTYPES:
        raise ValueError(f"dtype={dtype} must be float16, bfloat16 or float32")
    return _ext().read_kv(cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales, slots,
                          _DTYPES[dtype])


def attend_kv(
    q: torch.Tensor,
    cache: KVCache,
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    query_offsets: Optional[torch.Tensor] = None,
    max_query_len: Optional[int] = None,
    scale: Optional[float] = None,
    causal: bool = True,
) -> torch.Tensor:
    """softmax(scale q k^T) v of each query over its sequence's cached keys.

    q [tokens, q_heads, head_size], fp16 or bf16, q_heads a multiple of the
    cache's heads (query head h reads cache head h // (q_heads / heads)).
    Sequence b has ``seq_lens[b]`` keys and the queries
    ``query_offsets[b]:query_offsets[b + 1]`` (offsets that decrease anywhere
    give zeros for all); without query_offsets, one query
    a sequence. The queries are the last tokens of their sequence, their keys
    appended already: with ``causal``, query i of n sees ``seq_lens[b] - n + i
    + 1`` keys. A query that sees none gives 0, and so does one of no sequence
    (a captured step's places past its last token). ``max_query_len`` (the most
    queries a sequence has; default: all of them) picks kernels and changes no
    result beyond the order of its sums. scale: head_size ** -0.5 by default.
    """
    if max_query_len is None:
        max_query_len = 1 if query_offsets is None else max(1, q.shape[0])
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _ext().attend_kv(q, cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales,
                            block_tables, seq_lens, query_offsets, max_query_len, scale, causal)
