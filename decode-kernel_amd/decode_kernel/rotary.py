"""Rotary positions of queries and keys, of one or several axes.

What q and k go through between their projection and ``append_kv`` /
``attend_kv``: pair i of each head turns by ``positions[axis of i] *
frequencies[i]``. Text has one axis (``plan_kv_step``'s positions); images and
video have time, height and width, each with frequencies of its own.

    rotary = Rotary.from_base(128, 10000.0, sections=(16, 24, 24))   # once
    q, k = rotate_qk(q, k, positions, rotary)                        # once a layer

The reference has no counterpart (python/decode_kernel/__init__.py:32-83). Like
``gemv``, rotate_qk runs only through the HIP extension
(include/decode_kernel/dk_rotary.h).
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from ._native import ext as _ext

__all__ = ["Rotary", "rotate_qk"]


@dataclass
class Rotary:
    """Which elements of a head turn together, how fast, and by which axis."""

    frequencies: torch.Tensor             # fp32 [pairs]: radians a position
    axes: Optional[torch.Tensor] = None   # int32 [pairs]: the axis of each, or all 0
    adjacent: bool = False                # pairs (2i, 2i + 1), else (i, pairs + i)

    @classmethod
    def from_base(cls, rotary_size: int, base: float = 10000.0, sections: Optional[Sequence[int]] = None,
                  interleaved: bool = False, adjacent: bool = False,
                  device: torch.device | str = "cuda") -> "Rotary":
        """Frequencies ``base ** (-2 i / rotary_size)`` for the first rotary_size
        elements of a head.

        sections: how many of the rotary_size / 2 pairs turn by each axis, first
        the first axis' pairs, then the next's. interleaved: pair i turns by axis
        i % axes while that axis has pairs left among the first ``axes *
        sections[axis]``, and by the first axis otherwise, so that every axis has
        slow and fast pairs.
        """
        if rotary_size < 2 or rotary_size % 2:
            raise ValueError(f"rotary_size={rotary_size} must be even and at least 2")
        pairs = rotary_size // 2
        frequencies = float(base) ** (-torch.arange(pairs, dtype=torch.float64) * 2 / rotary_size)
        axes = None
        if sections is not None:
            if sum(sections) != pairs or min(sections) < 0:
                raise ValueError(f"sections={tuple(sections)} must add up to the {pairs} pairs")
            if interleaved:
                n = len(sections)
                order = [i % n if i < n * sections[i % n] else 0 for i in range(pairs)]
            else:
                order = [a for a, count in enumerate(sections) for _ in range(count)]
            axes = torch.tensor(order, dtype=torch.int32, device=device)
        return cls(frequencies.float().to(device), axes, adjacent)


def rotate_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary,
              inverse: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """q and k [tokens, heads, head_size] (fp16 or bf16), turned, as new tensors.

    positions: int32 or int64 [tokens], or [axes, tokens] where ``rotary`` names
    axes (a number outside of them counts as the nearest). The pair (a, b)
    becomes (a cos - b sin, a sin + b cos); elements past the rotary's pairs are
    copied. inverse turns back, which is also what the gradient of the results
    goes through. Angles are formed in 64 bits: a position in the millions is as
    exact as a small one. q and k may be slices of one projection. The two results
    share one allocation.
    """
    return _ext().rotate_qk(q, k, positions, rotary.frequencies, rotary.axes, rotary.adjacent, inverse)
