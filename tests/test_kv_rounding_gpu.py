"""What attention over the paged cache rounds, held against 64 bits closer
than tests/test_kv_gpu.py does. The bound, per output, with a = sum p |v| / sum p:

    half a step of the output's type + 2^-14 a + keys floor 127 top

* the rounding of the result;
* the fp32 of scores, weights and sums. A score's terms add up to about 10 in
  base 2 here, each rounded at 2^-24 of that a few times, and up to 2000 tiles
  of keys are added up, each rounded at 2^-24 of the sum: under 2^-14 in all.
  A weight goes into the second product as two fp16 parts, 2^-22 of it off;
* where those two parts end: a weight under `floor` of its row's largest is
  lost, times a value of the largest scale of its tile of 64 keys, `top`.
  2^-36 with few rows, 2^-30 with many (where one unit holds for tiles whose
  scales are within 2^6 of each other).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle
from test_kv_gpu import DTYPES, _cache, _dev, _half_step, _random_cache, _tables

pytestmark = pytest.mark.gpu

FEW, MANY = 2.0**-36, 2.0**-30


def _attend(q, host, tables, lens, new, dtype, floor, scale=None, top=None, causal=True, batch=1, heads=1):
    """Runs attend_kv on one batch and holds it against the bound; `top` is
    the largest value scale of tiles that have a say (default: of all). The
    sequences stand `batch` times in the call, and the heads `heads` times in
    the cache, so that each goes through one share of the work in one piece."""
    from decode_kernel import attend_kv

    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    many = np.concatenate([[0], np.cumsum(new * batch)]).astype(np.int32)
    q = _dev(q.astype(np.float32), DTYPES[dtype])
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    cache = _cache(*(np.tile(a, (1,) * (a.ndim - 1 - (a.ndim > 2)) + (heads,) + (1,) * (a.ndim > 2)) for a in host))
    got = attend_kv(q.repeat(batch, heads, 1), cache, _dev(np.tile(tables, (batch, 1))),
                    torch.tensor(lens * batch, dtype=torch.int32, device="cuda"), _dev(many), max(new), scale=scale, causal=causal)
    ref, spread = kv_oracle.attend(q.double().cpu().numpy(), *host, tables, lens, offsets, scale, causal)
    top = host[3].max() if top is None else top
    got = got.double().view(batch, q.shape[0], heads, q.shape[1], -1).cpu().numpy()
    ref, spread = ref[None, :, None], spread[None, :, None]
    bound = _half_step(ref, DTYPES[dtype]) + 2.0**-14 * spread + max(lens) * floor * 127 * top
    assert np.isfinite(got).all()
    err = np.abs(got - ref)
    off = err > bound
    assert not off.any(), f"{off.sum()} of {off.size} outputs off, worst {(err / bound).max():.2f} bounds, " \
                          f"first {np.argwhere(off)[:3].tolist()}"
    return got, ref


# Times a sequence and a head of it stand in a call, so that each wave (few
# rows) or workgroup (many) has an item whole.
WHOLE = {FEW: dict(batch=256, heads=8), MANY: dict(batch=32, heads=8)}


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("d,page,group", [(128, 16, 8), (64, 64, 3), (128, 128, 1)])
@pytest.mark.parametrize("new,floor", [([1, 1], FEW), ([9, 4], FEW), ([300, 129], MANY), ([200, 500], MANY)])
def test_results_are_as_exact_as_their_rounding(new, floor, d, page, group, dtype):
    # Prompts from their first token on: rows of two and three keys show a
    # weight's rounding whole.
    rng = np.random.default_rng(d + page)
    new = [n * 8 // group if floor == MANY else n for n in new]
    lens = list(new) if floor == MANY else [70, 700]
    tables, pages = _tables(rng, lens, page)
    host = _random_cache(rng, pages, page, 2, d)
    _attend(rng.standard_normal((sum(new), 2 * group, d)), host, tables, lens, new, dtype, floor)


def _tile_scales(tile_scales, page, zero=(), heads=1, d=64):
    """Pages in order whose value scale is given tile by tile of 64 keys; in
    tiles `zero` all codes are 0."""
    rng = np.random.default_rng(len(tile_scales))
    each = max(64 // page, 1)
    scales = np.repeat(np.asarray(tile_scales, np.float64), each)[:: max(page // 64, 1)]
    host = list(_random_cache(rng, len(scales), page, heads, d))
    host[1] = np.clip(np.rint(60 + 30 * rng.standard_normal(host[1].shape)), -127, 127).astype(np.int8)
    host[3] = np.repeat(scales[:, None], heads, 1).astype(np.float32)
    for t in zero:
        host[1][t * each * 64 // max(page, 64): (t + 1) * each * 64 // max(page, 64)] = 0
    return rng, host, np.arange(len(scales), dtype=np.int32)[None], len(scales) * page


ONE = 1 / 38
TILES = {
    "34": [ONE] * 60 + [1e-34 / 127] + [ONE] * 5,
    "37": [ONE] * 60 + [1e-37 / 127] + [ONE] * 5,
    "both": [ONE] * 40 + [1e-34 / 127] + [ONE] * 8 + [1e-37 / 127] + [ONE] * 3,
    "last": [ONE] * 60 + [1e-34 / 127] * 2,
    "first": [1e-34 / 127] * 3 + [ONE] * 20,
    "first37": [1e-37 / 127] * 3 + [ONE] * 20,
    "large": [2000.0] * 20 + [1e-34 / 127] * 2 + [2000.0],
    "down": list(10.0 ** -np.arange(0, 36, 1.5)),
    "up": list(10.0 ** -np.arange(0, 36, 1.5))[::-1],
    "steps": [ONE, ONE * 40, ONE / 40, ONE * 900, ONE / 900, ONE * 20000, ONE / 20000] * 4,
    "tiny": [1e-34 / 127] * 20,
}


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,floor", [(1, FEW), (20, FEW), (140, MANY), (256, MANY)])
@pytest.mark.parametrize("which", sorted(TILES))
def test_value_scales_of_any_ratio(which, new, floor, page):
    # bf16 values reach down to 1e-38: pages of such values among ordinary
    # ones, whichever comes first.
    rng, host, tables, n = _tile_scales(TILES[which], page)
    q = rng.standard_normal((new, 1, 64))
    _attend(q, host, tables, [n], [new], "bf16", floor, causal=False)
    _attend(q, host, tables, [n], [new], "bf16", floor, causal=False, **WHOLE[floor])


@pytest.mark.parametrize("new,floor", [(1, FEW), (140, MANY)])
@pytest.mark.parametrize("large", [ONE, 1e10])
@pytest.mark.parametrize("tiny", [1e-20, 1e-30])
def test_small_values_after_zeros_on_large_pages(tiny, large, new, floor):
    # Nothing has been summed when the scales fall: what follows is all there is.
    rng, host, tables, n = _tile_scales([large] * 6 + [tiny] * 6 + [large] * 3, 16, zero=[*range(6), 12, 13, 14])
    got, ref = _attend(rng.standard_normal((new, 1, 64)), host, tables, [n], [new], "bf16", floor, causal=False, top=tiny, **WHOLE[floor])
    assert np.abs(ref).max() > tiny and np.abs(got).max() > tiny


def _sink(n, delta, first, d=64, page=16):
    """One key that takes nearly all weight and has value 0, and n - 1 keys
    2^-delta below it. Its page's value scale is `first` times the others'."""
    rng = np.random.default_rng(n + int(delta))
    count = -(-n // page)
    k = np.zeros((count, page, 1, d), np.int8)
    k[:, :, 0, 0] = rng.integers(-3, 4, (count, page))
    k[0, 0, 0, 0] = 127
    v = np.clip(np.rint(60 + 40 * rng.standard_normal((count, page, 1, d))), -127, 127).astype(np.int8)
    v[0] = 0
    ks, vs = np.full((count, 1), 1 / 127, np.float32), np.ones((count, 1), np.float32)
    vs[:max(64 // page, 1)] = first  # the whole first tile
    v[:max(64 // page, 1)] = 0
    tables = rng.permutation(count).astype(np.int32)
    place = np.argsort(tables)
    host = [a[place] for a in (k, v, ks, vs)]
    return host, tables[None], delta * np.log(2.0)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("n,delta", [(20000, 18), (20000, 24), (20000, 26), (131070, 24), (131070, 26)])
@pytest.mark.parametrize("first", [1.0, 50.0])
def test_small_weights_beside_a_sink_few_rows(first, n, delta, dtype):
    host, tables, scale = _sink(n, delta, first)
    q = np.zeros((1, 2, 64))
    q[..., 0] = 1
    _attend(q, host, tables, [n], [1], dtype, FEW, scale=scale, top=1.0, **WHOLE[FEW])
    _attend(q, host, tables, [n], [1], dtype, FEW, scale=scale, top=1.0)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("n,delta", [(20000, 18), (20000, 20), (20000, 24)])
@pytest.mark.parametrize("first", [1.0, 50.0, 1 / 50])
def test_small_weights_beside_a_sink_many_rows(first, n, delta, dtype):
    host, tables, scale = _sink(n, delta, first)
    q = np.zeros((140, 1, 64))
    q[..., 0] = 1
    _attend(q, host, tables, [n], [140], dtype, MANY, scale=scale, top=1.0, **WHOLE[MANY])


@pytest.mark.parametrize("new,floor", [(2, FEW), (140, MANY)])
@pytest.mark.parametrize("scales", [[ONE] * 6 + [1e-34 / 127] * 6, [1e-34 / 127] * 6 + [ONE] * 6,
                                    [ONE] * 5 + [1e-34 / 127] * 5 + [ONE] * 5 + [1e-34 / 127] * 5])
def test_rows_that_look_past_large_values(scales, new, floor):
    # Every other row has all its weight on the pages of small values; the large
    # ones weigh 2^-200 there, and nothing of them is left.
    rng, host, tables, n = _tile_scales(scales, 16)
    small = np.repeat(np.asarray(scales) < 1e-30, 4)
    host[0][:] = 0
    host[0][..., 0] = np.where(small, 100, -100)[:, None, None]
    host[0][..., 1] = rng.integers(-100, 101, host[0].shape[:-1])
    host[2][:] = 0.01
    q = np.zeros((new, 1, 64))
    q[:, 0, 0] = np.where(np.arange(new) % 2, 100, -100) * np.log(2.0)
    q[:, 0, 1] = 1
    got, ref = _attend(q, host, tables, [n], [new], "bf16", floor, scale=1.0, causal=False, top=0.0, **WHOLE[floor])
    assert np.abs(ref[:, 1::2]).max() < 1e-30 and np.abs(ref[:, ::2]).min() > 0.1
