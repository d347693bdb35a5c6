"""The paged 8-bit key/value cache on the GPU against oracle/kv_oracle.py.

Planning is compared exactly, appending bit for bit with the definition in
fp32 (codes and scales), reading bit for bit, attention with the definition
in 64 bits. The attention's bound, per output, with a = sum p |v| / sum p:

    half a step of the output's type + (2^-11 + 1e-4) a + keys 2^-25 max |v|

which is the rounding of the result, that of the weights p to fp16 before
the second product (2^-11 each, and 2^-25 below fp16's normal range), and the
fp32 of the scores: a score of size s is off by a few 2^-24 s, its weight
relatively by that, under 1e-4 for the |s| < 200 here.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_oracle

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def _cache(codes_k, codes_v, ks, vs):
    from decode_kernel import KVCache

    kc, vc = kv_oracle.to_device_layout(codes_k, codes_v)
    return KVCache(_dev(kc), _dev(vc), _dev(ks), _dev(vs))


def _back(cache):
    k, v = kv_oracle.from_device_layout(cache.k_codes.cpu().numpy(), cache.v_codes.cpu().numpy())
    return k, v, cache.k_scales.cpu().numpy(), cache.v_scales.cpu().numpy()


def _random_cache(rng, pages, page, heads, d, k_std=1.0, v_std=1.0, spread=0.3):
    codes = lambda: np.clip(np.rint(rng.standard_normal((pages, page, heads, d)) * 40), -127, 127).astype(np.int8)  # noqa: E731
    scales = lambda std: (std / 40 * np.exp(spread * rng.standard_normal((pages, heads)))).astype(np.float32)  # noqa: E731
    return codes(), codes(), scales(k_std), scales(v_std)


# ------------------------------------------------------------------- planning
def _plan_case(seed, b, page, width, held_hi, added, free, tokens=None):
    rng = np.random.default_rng(seed)
    held = rng.integers(0, held_hi + 1, b).astype(np.int32)
    added = np.asarray([added(rng) for _ in range(b)], np.int32)
    tables = np.full((b, width), -1, np.int32)
    ids = rng.permutation(b * width + free + 5).astype(np.int32)
    for i in range(b):
        n = min(-(-int(held[i]) // page), width)
        tables[i, :n] = ids[i * width: i * width + n]
    free_pages = ids[b * width: b * width + free + 5]
    total = int(np.maximum(added, 0).sum()) if tokens is None else tokens
    return tables, held, added, free_pages, free, page, total


PLANS = [
    # requests, page, table width, held up to, added, free pages, tokens
    (1, 16, 4, 0, lambda r: 1, 3, None),
    (1, 16, 4, 17, lambda r: 40, 9, None),
    (5, 32, 6, 100, lambda r: int(r.integers(0, 60)), 30, None),
    (7, 64, 9, 200, lambda r: int(r.integers(-3, 200)), 60, None),
    (200, 16, 20, 300, lambda r: 1, 300, None),
    (300, 128, 5, 500, lambda r: int(r.integers(0, 9)), 700, None),
    (4096, 16, 3, 40, lambda r: int(r.integers(0, 2)), 5000, None),
    (3, 16, 70, 0, lambda r: 1000, 500, None),
    (6, 16, 10, 60, lambda r: 30, 4, None),        # too few free pages
    (6, 16, 10, 60, lambda r: 30, 0, None),        # none at all
    (5, 16, 3, 40, lambda r: 30, 40, None),        # past the tables' end
    (5, 16, 12, 40, lambda r: 30, 40, 77),         # fewer places than tokens
    (5, 16, 12, 40, lambda r: 30, 40, 333),        # more
    (5, 16, 12, 40, lambda r: 0, 40, 9),           # nothing new
    (5, 16, 12, 40, lambda r: 10, 40, 0),          # no places
    (0, 16, 4, 0, lambda r: 1, 3, 5),              # no requests
    (4, 16, 0, 40, lambda r: 3, 10, None),         # no table
    (3, 16, 10, 40, lambda r: 2**30, 40, 50),      # sums past 31 bits
]


@pytest.mark.parametrize("i", range(len(PLANS)))
def test_plan(i):
    from decode_kernel import plan_kv_step

    b, page, width, held_hi, added, free, tokens = PLANS[i]
    tables, held, add, free_pages, count, page, total = _plan_case(i, b, page, width, held_hi, added, free, tokens)
    want = kv_oracle.plan(tables, held, add, free_pages, count, page, total)
    t = _dev(tables)
    args = (t, _dev(held), _dev(add), _dev(free_pages), torch.tensor([count], dtype=torch.int32, device="cuda"), page, total)
    for _ in range(2):  # a function of its inputs: the same again
        got = plan_kv_step(*args)
        np.testing.assert_array_equal(t.cpu().numpy(), want[0])
        for g, w in zip(got[:4], want[1:5]):
            np.testing.assert_array_equal(g.cpu().numpy(), w)
        assert got.free_count.tolist() == [want[5]]
    assert got.slots.dtype == torch.int64 and got.seq_lens.dtype == torch.int32


def test_plan_free_count_past_the_list():
    # A count larger than the list is cut to it: nothing is read past its end.
    from decode_kernel import plan_kv_step

    t = torch.full((1, 4), -1, dtype=torch.int32, device="cuda")
    one = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    got = plan_kv_step(t, one(0), one(33), torch.arange(5, 7, dtype=torch.int32, device="cuda"), one(1000), 16, 33)
    assert t.tolist() == [[6, 5, -1, -1]]
    assert got.slots.tolist() == list(range(96, 112)) + list(range(80, 96)) + [-1]
    assert got.free_count.tolist() == [997] and got.seq_lens.tolist() == [33]


# ------------------------------------------------------------------ appending
def _append_case(seed, page, heads, d, spans, pages=None, scale=1.0):
    """spans: (first offset in the page, tokens) of each request; pages in a
    random order. Returns slots and x."""
    rng = np.random.default_rng(seed)
    need = sum(-(-(o + n) // page) for o, n in spans)
    pages = need + 3 if pages is None else pages
    ids = list(rng.permutation(pages))
    slots = []
    for off, n in spans:
        mine = [ids.pop() for _ in range(-(-(off + n) // page))]
        slots += [int(mine[t // page]) * page + t % page for t in range(off, off + n)]
    x = [(scale * rng.standard_normal((len(slots), heads, d))).astype(np.float32) for _ in range(2)]
    return rng, pages, np.array(slots, np.int64), x


SPANS = [
    [(0, 1)], [(5, 1)], [(15, 1)], [(0, 16)], [(3, 13)], [(7, 50)],
    [(0, 1), (1, 1), (9, 1), (15, 2)], [(0, 200), (4, 1), (0, 33), (11, 70)],
]


def _check_append(cache, before, x, xt, slots):
    from decode_kernel import append_kv

    want = [a.copy() for a in before]
    kv_oracle.append(want[0], want[2], x[0], slots)
    kv_oracle.append(want[1], want[3], x[1], slots)
    sd = _dev(slots)
    for _ in range(2):  # a step made twice leaves the same
        append_kv(cache, xt[0], xt[1], sd)
        for g, w in zip(_back(cache), want):
            np.testing.assert_array_equal(g, w)
    return want


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("page,heads,d", [(16, 3, 128), (32, 1, 64), (64, 2, 128), (128, 5, 64), (128, 2, 128)])
@pytest.mark.parametrize("spans", range(len(SPANS)))
def test_append(spans, page, heads, d, dtype):
    rng, pages, slots, x = _append_case(spans, page, heads, d, SPANS[spans])
    before = _random_cache(rng, pages, page, heads, d)
    xt = [_dev(a, DTYPES[dtype]) for a in x]
    x = [a.float().cpu().numpy() for a in xt]
    want = _check_append(_cache(*before), before, x, xt, slots)
    # The definition in 64 bits: a new value is half a step of its page away.
    for codes, scales, xs in ((want[0], want[2], x[0]), (want[1], want[3], x[1])):
        step = scales[slots // page][:, :, None].astype(np.float64)
        off = np.abs(kv_oracle.read(codes, scales, slots) - xs)
        assert (off <= step * (0.5 + 1e-5)).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("page,heads,d", [(16, 2, 64), (32, 1, 128), (64, 2, 128), (128, 1, 64), (128, 2, 128)])
def test_append_many_tokens(page, heads, d, dtype):
    # Past 256 tokens: long runs on all waves of a workgroup, runs of one token
    # among them, tokens without a slot inside, at a start and at an end.
    spans = [(0, 300), (5, 1), (page - 1, 1), (9, page + 30), (0, 1), (3, 2), (0, page), (14, 5), (1, 200)]
    rng, pages, slots, x = _append_case(page + d, page, heads, d, spans)
    assert len(slots) > 256
    for lo, hi in ((7, 9), (297, 301), (350, 351), (len(slots) - 4, len(slots) - 1)):
        slots[lo:hi] = -1
    before = _random_cache(rng, pages, page, heads, d)
    xt = [_dev(a, DTYPES[dtype]) for a in x]
    _check_append(_cache(*before), before, [a.float().cpu().numpy() for a in xt], xt, slots)


def test_append_scale_kept_and_grown():
    # One request's tokens one by one: scales only grow, and each stored value
    # is within half a step of the scale at its writing plus half a step for
    # each time the scale grew since.
    from decode_kernel import KVCache, append_kv, read_kv

    page, heads, d, n = 32, 2, 128, 70
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((n, heads, d)) * np.exp(rng.standard_normal((n, 1, 1)))).astype(np.float16)
    cache = KVCache.empty(3, heads, d, page)
    ref = [np.zeros((3, page, heads, d), np.int8), np.zeros((3, heads), np.float32)]
    grew = np.zeros((n, heads))
    xd = _dev(x)
    for t in range(n):
        append_kv(cache, xd[t:t + 1], xd[t:t + 1], torch.tensor([t], device="cuda"))
        old = ref[1].copy()
        kv_oracle.append(*ref, x[t:t + 1].astype(np.float32), np.array([t]))
        if t % page:
            grew[t // page * page: t] += (ref[1] > old)[t // page]
    got = _back(cache)
    for k in (0, 1):
        np.testing.assert_array_equal(got[k], ref[0])
        np.testing.assert_array_equal(got[k + 2], ref[1])
    k, _ = read_kv(cache, torch.arange(n, device="cuda"), torch.float32)
    step = ref[1][np.arange(n) // page]
    err = np.abs(k.cpu().numpy() - x.astype(np.float32)).max(-1)
    assert (err <= step * (0.5 + 0.5 * grew + 1e-4)).all()


def test_append_skips_slots_outside_the_cache():
    page, heads, d = 16, 2, 64
    rng, pages, slots, x = _append_case(5, page, heads, d, [(2, 40), (0, 9)])
    slots[10:13] = -1
    slots[30] = pages * page          # one past the end
    slots[31] = 2**40
    slots[32] = -(2**40)
    before = _random_cache(rng, pages, page, heads, d)
    xt = [_dev(a, torch.float16) for a in x]
    _check_append(_cache(*before), before, [a.float().cpu().numpy() for a in xt], xt, slots)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_non_finite(bad):
    # The page's values for that head become NaN; nothing else changes.
    from decode_kernel import append_kv, read_kv

    page, heads, d = 16, 3, 128
    rng, pages, slots, x = _append_case(6, page, heads, d, [(4, 30)])
    before = _random_cache(rng, pages, page, heads, d)
    cache = _cache(*before)
    xt = [_dev(a, torch.float16) for a in x]
    xt[0][3, 1, 77] = bad
    xt[1][20, 2, 5] = bad
    append_kv(cache, *xt, _dev(slots))
    k, v = read_kv(cache, _dev(slots), torch.float32)
    hit = lambda t: slots // page == slots[t] // page  # noqa: E731
    for got, t, h in ((k, 3, 1), (v, 20, 2)):
        nan = torch.isnan(got).cpu().numpy()
        want = np.zeros_like(nan)
        want[hit(t), h] = True
        np.testing.assert_array_equal(nan, want)


def test_append_zeros_and_tiny():
    # All zeros, and values whose scale is under 2^-126 (bf16 alone has them).
    from decode_kernel import KVCache, append_kv

    page, heads, d = 16, 2, 64
    x = torch.zeros(20, heads, d, dtype=torch.bfloat16, device="cuda")
    x[:, 1] = 1e-37
    cache = KVCache.empty(2, heads, d, page)
    append_kv(cache, x, x, torch.arange(20, device="cuda"))
    k, v, ks, vs = _back(cache)
    assert not k.any() and not v.any()
    assert (ks[:, 0] == 0).all() and (ks[:, 1] == np.float32(x[0, 1, 0].item()) * (np.float32(1) / np.float32(127))).all()
    np.testing.assert_array_equal(ks, vs)


@pytest.mark.parametrize("how", ["fused", "odd", "transposed", "shifted"])
def test_append_and_attend_strides(how):
    # A slice of a fused projection is read in place, odder ones are copied.
    from decode_kernel import append_kv, attend_kv

    page, heads, d, n = 16, 2, 64, 37
    rng = np.random.default_rng(8)
    before = _random_cache(rng, 4, page, heads, d)
    base = torch.from_numpy(rng.standard_normal((3, n, heads, d)).astype(np.float16)).cuda()
    if how == "fused":
        rows = torch.cat([b.reshape(n, -1) for b in base], 1)
        views = [rows[:, i * heads * d:(i + 1) * heads * d].view(n, heads, d) for i in range(3)]
    elif how == "odd":
        wide = torch.zeros(n, heads, d + 3, dtype=torch.float16, device="cuda")
        views = []
        for b in base:
            w = wide.clone()
            w[:, :, :d] = b
            views.append(w[:, :, :d])
    elif how == "transposed":
        views = [b.permute(2, 1, 0).contiguous().permute(2, 1, 0) for b in base]
    else:
        views = []
        for b in base:
            flat = torch.zeros(b.numel() + 1, dtype=torch.float16, device="cuda")
            flat[1:] = b.reshape(-1)
            views.append(flat[1:].view(n, heads, d))
    slots = torch.arange(n, device="cuda")
    tables = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    offs = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    outs = []
    for q, k, v in (base, views):
        cache = _cache(*before)
        append_kv(cache, k, v, slots)
        outs.append((_back(cache), attend_kv(q, cache, tables, lens, offs, n)))
    for a, b in zip(outs[0][0], outs[1][0]):
        np.testing.assert_array_equal(a, b)
    assert torch.equal(outs[0][1], outs[1][1])


# -------------------------------------------------------------------- reading
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,heads,d,n", [(16, 3, 128, 1), (16, 8, 128, 77), (32, 1, 64, 64), (64, 2, 128, 130), (128, 5, 64, 300)])
def test_read(page, heads, d, n, dtype):
    from decode_kernel import read_kv

    rng = np.random.default_rng(n)
    pages = 9
    host = _random_cache(rng, pages, page, heads, d)
    cache = _cache(*host)
    orders = [np.arange(n) + 3, rng.integers(0, pages * page, n), rng.permutation(pages * page)[:n]]
    orders[1][::5] = -1
    orders[1][n // 2] = pages * page
    for slots in orders:
        got = read_kv(cache, _dev(slots.astype(np.int64)), dtype)
        for g, codes, scales in zip(got, host[:2], host[2:]):
            # code * scale is exact in 64 bits and rounded once to fp32; the
            # halves round that again, as torch does here.
            want = torch.from_numpy(kv_oracle.read(codes, scales, slots).astype(np.float32)).to(dtype)
            assert torch.equal(g.cpu(), want)


# ------------------------------------------------------------------ attention
def _tables(rng, lens, page, width=None, extra=3):
    count = [-(-n // page) for n in lens]
    width = max(max(count, default=0), 1) + 1 if width is None else width
    pages = sum(count) + extra
    ids = list(rng.permutation(pages))
    tables = np.full((len(lens), width), -1, np.int32)
    for b, c in enumerate(count):
        tables[b, :c] = [ids.pop() for _ in range(c)]
    return tables, pages


def _half_step(ref, dtype):
    mant, low = (10, -24) if dtype == torch.float16 else (7, -133)
    e = np.floor(np.log2(np.maximum(np.abs(ref), 1e-300)))
    return 0.5 * np.exp2(np.maximum(e - mant, low))


def _check(got, ref, spread, keys, vmax, dtype, label=""):
    got = got.float().cpu().numpy().astype(np.float64)
    live = ~np.isnan(ref)
    bound = _half_step(ref, dtype) + (2.0**-11 + 1e-4) * spread + keys * 2.0**-25 * vmax
    err = np.abs(got - ref)
    bad = live & ~(err <= bound)
    assert not bad.any(), f"{label}: {bad.sum()} outputs off, first {np.argwhere(bad)[:3].tolist()}, " \
                          f"worst {np.nanmax(np.where(live, err / bound, 0)):.2f} bounds"


def _attend_case(seed, lens, new, heads, group, d, page, dtype, causal=True, host=None, tables=None,
                 max_query_len="exact", q_std=1.0, **kw):
    """new: queries of each sequence, or None for the form without offsets."""
    from decode_kernel import attend_kv

    rng = np.random.default_rng(seed)
    made, pages = _tables(rng, lens, page)
    tables = made if tables is None else tables
    host = _random_cache(rng, pages, page, heads, d, **kw) if host is None else host
    cache = _cache(*host)
    counts = [1] * len(lens) if new is None else new
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = _dev((q_std * rng.standard_normal((offsets[-1], heads * group, d))).astype(np.float32), DTYPES[dtype])
    most = max(counts, default=1) if max_query_len == "exact" else max_query_len
    lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = attend_kv(q, cache, _dev(tables), lens_d, None if new is None else _dev(offsets),
                    None if most is None else max(1, most), causal=causal)
    assert got.shape == q.shape and got.dtype == q.dtype
    ref, spread = kv_oracle.attend(q.float().cpu().numpy(), *host, tables, lens, offsets, d**-0.5, causal)
    vmax = 127 * np.abs(host[3][np.isfinite(host[3])]).max()
    _check(got, ref, spread, max(lens, default=0), vmax, DTYPES[dtype])
    return got, ref


@pytest.mark.parametrize("length", [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 4097])
@pytest.mark.parametrize("page,d", [(16, 128), (32, 64), (64, 128), (128, 64)])
def test_attend_one_sequence(length, page, d):
    _attend_case(length, [length], None, 2, 4, d, page, "fp16")


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("heads,group", [(1, 1), (3, 2), (2, 5), (1, 16), (1, 17), (2, 40), (8, 8)])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_attend_heads(heads, group, page, dtype):
    _attend_case(heads * group, [5, 700, 0, 129, 64], None, heads, group, 128, page, dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b", [1, 7, 64, 255, 256, 257, 600])
def test_attend_ragged_batch(b, d):
    rng = np.random.default_rng(b)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(500), b))]
    lens[b // 2] = 0
    lens[-1] = 1500
    _attend_case(b, lens, None, 1, 3, d, 16, "bf16")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("d,page,dtype", [(128, 16, "fp16"), (64, 64, "bf16"), (128, 128, "bf16"), (64, 32, "fp16")])
def test_attend_several_queries(d, page, dtype, group, causal):
    # From one query to a prompt; sequences of only new tokens, none, and more
    # queries than keys (rows that see nothing).
    lens = [300, 40, 64, 0, 5, 130, 333, 1, 65]
    new = [1, 40, 7, 2, 9, 0, 129, 1, 64]
    _attend_case(group, lens, new, 2, group, d, page, dtype, causal)


@pytest.mark.parametrize("max_query_len", [1, 5, 1000, None])
def test_attend_max_query_len_only_picks_kernels(max_query_len):
    _attend_case(11, [200, 500, 90], [3, 150, 1], 2, 4, 128, 32, "fp16", max_query_len=max_query_len)


@pytest.mark.parametrize("new", [33, 127, 128, 129, 500])
@pytest.mark.parametrize("group,page", [(1, 16), (4, 64), (8, 128)])
def test_attend_prompt(new, group, page):
    # A prompt alone, and on top of a context that no tile divides.
    _attend_case(new, [new, new + 77], [new, new], 1, group, 128, page, "fp16")


def test_attend_long_sequence_with_short_ones():
    _attend_case(1, [20000, 3, 0, 64, 1], None, 2, 8, 128, 64, "fp16")


@pytest.mark.parametrize("b,heads", [(1, 1), (63, 1), (65, 2), (64, 4), (200, 1), (255, 1), (256, 1), (257, 1), (129, 2)])
@pytest.mark.parametrize("longest", [1, 63, 448, 449, 960, 961])
def test_attend_items_of_one_workgroup(b, heads, longest):
    # To 256 items of a few tiles each (448, 960 keys: the last that make two
    # shares' worth for eight waves), and just past that; idle ones among them.
    rng = np.random.default_rng(b)
    lens = [int(x) for x in rng.integers(0, longest + 1, b)]
    lens[b // 3] = longest
    _attend_case(b, lens, [int(x) for x in rng.integers(0, 3, b)], heads, 2, 64 if b % 2 else 128, 32, "fp16")


@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("d,page,dtype", [(128, 16, "bf16"), (64, 64, "fp16"), (128, 128, "fp16"), (64, 32, "bf16")])
def test_attend_several_queries_beside_a_long_sequence(d, page, dtype, group):
    # The long one has the shares cut across the short ones' items.
    lens = [300, 40, 3001, 64, 0, 5, 130, 333, 1, 65]
    new = [1, 16, 1, 7, 2, 9, 0, 15, 1, 12]
    _attend_case(group, lens, new, 2, group, d, page, dtype)


@pytest.mark.parametrize("new", [None, [90, 3]])
@pytest.mark.parametrize("scale", [-0.09, 0.0, 0.5])
def test_attend_scale(new, scale):
    # Any factor: a negative one turns the scores round, 0 takes the mean.
    from decode_kernel import attend_kv

    rng = np.random.default_rng(12)
    lens, heads, group, d, page = [150, 700], 2, 3, 64, 32
    tables, pages = _tables(rng, lens, page)
    host = _random_cache(rng, pages, page, heads, d)
    counts = new or [1, 1]
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = _dev(rng.standard_normal((offsets[-1], heads * group, d)).astype(np.float16))
    got = attend_kv(q, _cache(*host), _dev(tables), _dev(np.array(lens, np.int32)),
                    None if new is None else _dev(offsets), max(counts), scale=scale)
    ref, spread = kv_oracle.attend(q.float().cpu().numpy(), *host, tables, lens, offsets, scale, True)
    _check(got, ref, spread, max(lens), 127 * host[3].max(), torch.float16)


@pytest.mark.parametrize("new", [None, [100]])
def test_attend_zero_pages(new):
    # Pages whose scales are 0: their keys score 0, their values add nothing.
    rng = np.random.default_rng(13)
    lens, page = [230], 16
    tables, pages = _tables(rng, lens, page)
    host = _random_cache(rng, pages, page, 2, 128)
    host[2][tables[0, 3]] = 0
    host[3][tables[0, :9]] = 0
    _attend_case(13, lens, new, 2, 2, 128, page, "fp16", host=host, tables=tables)
    host[3][:] = 0
    got, _ = _attend_case(13, lens, new, 2, 2, 128, page, "fp16", host=host, tables=tables)
    assert not got.any()


def test_attend_queries_that_belong_to_nobody():
    # Offsets that leave queries out at the end, and ones that are no offsets:
    # what is in range is right, nothing else is touched or read.
    from decode_kernel import attend_kv

    rng = np.random.default_rng(14)
    lens = [100, 60]
    tables, pages = _tables(rng, lens, 16)
    host = _random_cache(rng, pages, 16, 1, 64)
    q = _dev(rng.standard_normal((50, 2, 64)).astype(np.float16))
    lens_d = _dev(np.array(lens, np.int32))
    for offsets, n in (([0, 3, 40], 40), ([0, 1, 2], 2)):
        got = attend_kv(q, _cache(*host), _dev(tables), lens_d, _dev(np.array(offsets, np.int32)), 37)
        ref, spread = kv_oracle.attend(q.float().cpu().numpy(), *host, tables, lens, offsets, 0.125, True)
        assert np.isnan(ref[n:]).all()
        _check(got[:n], ref[:n], spread[:n], 100, 127 * host[3].max(), torch.float16)
    wild = _dev(np.array([-5, 2**30, -(2**31)], np.int32))
    attend_kv(q, _cache(*host), _dev(tables), _dev(np.array([-7, 2**31 - 1], np.int32)), wild, 50)
    torch.cuda.synchronize()


def test_attend_sharp_scores():
    # Scores of some hundred apart: one key takes all, maxima move often.
    _attend_case(2, [3000, 100], None, 2, 4, 128, 16, "fp16", q_std=12.0)
    _attend_case(3, [300, 260], [70, 3], 2, 4, 128, 16, "fp16", q_std=12.0)


@pytest.mark.parametrize("new", [None, [90, 64]])
def test_attend_scales_of_every_size(new):
    # Page scales over four decades: weights are rounded relative to their own
    # page's values, not to the largest in sight.
    _attend_case(4, [900, 64], new, 2, 4, 128, 16, "fp16", spread=2.0, k_std=0.05)


@pytest.mark.parametrize("new", [None, [3, 40, 1]])
def test_attend_tiny_and_huge_queries(new):
    # bf16 queries whose size no fp16 holds, and an all-zero row.
    from decode_kernel import attend_kv

    rng = np.random.default_rng(5)
    lens, heads, group, d, page = [100, 300, 64], 2, 4, 128, 32
    tables, pages = _tables(rng, lens, page)
    host = _random_cache(rng, pages, page, heads, d)
    counts = new or [1] * 3
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = _dev(rng.standard_normal((offsets[-1], heads * group, d)).astype(np.float32)).bfloat16()
    for factor in (2.0**100, 2.0**-110, 0.0):
        qf = q * factor
        scale = d**-0.5 / factor if factor else 1.0
        if not np.isfinite(np.float32(scale)):
            continue
        got = attend_kv(qf, _cache(*host), _dev(tables), _dev(np.array(lens, np.int32)),
                        None if new is None else _dev(offsets), max(counts), scale=scale)
        ref, spread = kv_oracle.attend(qf.double().cpu().numpy(), *host, tables, lens, offsets, scale, True)
        _check(got, ref, spread, max(lens), 127 * host[3].max(), torch.bfloat16, f"{factor}")


@pytest.mark.parametrize("new", [None, [5, 70, 40]])
def test_attend_pages_that_are_not_there(new):
    # -1 or an id past the cache in the middle of a table: keys not seen.
    rng = np.random.default_rng(6)
    lens, page = [300, 500, 130], 16
    tables, pages = _tables(rng, lens, page)
    tables[0, 3] = -1
    tables[1, 0:9] = -1
    tables[1, 20] = pages + 5
    tables[1, 21] = 2**31 - 1
    tables[2, :] = -1  # nothing at all: zeros
    host = _random_cache(rng, pages, page, 2, 64)
    got, ref = _attend_case(6, lens, new, 2, 3, 64, page, "fp16", host=host, tables=tables)
    assert not got[-1].any()


@pytest.mark.parametrize("new", [None, [40, 65, 3]])
def test_attend_ignores_what_no_query_sees(new):
    # NaN and infinite scales on pages of no sequence, and table entries past
    # the sequence's end that name them.
    rng = np.random.default_rng(7)
    lens, page = [70, 130, 16], 16
    tables, pages = _tables(rng, lens, page, extra=6)
    host = _random_cache(rng, pages, page, 2, 128)
    unused = np.setdiff1d(np.arange(pages), tables)
    host[2][unused] = np.nan
    host[3][unused[::2]] = np.inf
    host[3][unused[1::2]] = np.nan
    for b, n in enumerate(lens):
        tables[b, -(-n // page):] = unused[b]
    _attend_case(7, lens, new, 2, 3, 128, page, "fp16", host=host, tables=tables)


@pytest.mark.parametrize("which,bad", [(2, np.nan), (3, np.nan), (3, np.inf)])
@pytest.mark.parametrize("n", [6, 100])
def test_attend_non_finite_page(which, bad, n):
    # Exactly the rows that see a page whose scale is not finite are not either.
    from decode_kernel import attend_kv

    rng = np.random.default_rng(8)
    length, page, heads, group, d = 200, 16, 2, 2, 64
    tables, pages = _tables(rng, [length], page)
    host = _random_cache(rng, pages, page, heads, d)
    col = (length - 3) // page  # its first tokens' queries do not see all of it
    host[which][tables[0, col], 1] = bad
    q = _dev(rng.standard_normal((n, heads * group, d)).astype(np.float16))
    got = attend_kv(q, _cache(*host), _dev(tables), torch.tensor([length], dtype=torch.int32, device="cuda"),
                    torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
    sees = (length - n + np.arange(n)) >= col * page
    off = ~torch.isfinite(got).cpu().numpy()
    want = np.zeros_like(off)
    want[sees, group:] = True
    np.testing.assert_array_equal(off, want)


@pytest.mark.parametrize("n", [1, 50])
def test_attend_offsets_past_32_bits(n):
    # Pages whose codes lie past 4 GiB, and their token slots past 2^31 bytes.
    from decode_kernel import KVCache, append_kv, attend_kv, read_kv

    page, heads, d = 128, 8, 128
    pages = (9 << 29) // (page * heads * d)  # 4.5 GiB of keys
    cache = KVCache.empty(pages, heads, d, page)
    rng = np.random.default_rng(9)
    ids = np.array([pages - 1, 0, pages - 2, pages // 2 + 1], np.int32)
    length = 4 * page - 5
    x = [_dev(rng.standard_normal((length, heads, d)).astype(np.float16)) for _ in range(2)]
    slots = torch.from_numpy(np.repeat(ids.astype(np.int64) * page, page) + np.tile(np.arange(page), 4)).cuda()[:length]
    append_kv(cache, *x, slots)
    k, v = read_kv(cache, slots, torch.float32)
    for got, want in ((k, x[0]), (v, x[1])):
        assert (got - want.float()).abs().max() < 0.5 * 6.0 / 127 * 1.01  # amax under 6
    q = _dev(rng.standard_normal((n, heads, d)).astype(np.float16))
    got = attend_kv(q, cache, _dev(ids[None]), torch.tensor([length], dtype=torch.int32, device="cuda"),
                    torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
    s = torch.einsum("qhd,khd->hqk", q.float(), k) * d**-0.5
    s = s.masked_fill(torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda")[:, None], -np.inf)
    want = torch.einsum("hqk,khd->qhd", s.softmax(-1), v)
    assert (got.float() - want).abs().max() < 2e-3


# ------------------------------------------------- steps, streams and graphs
def _step_state(seed, b=5, heads=2, group=4, d=128, page=16):
    from decode_kernel import KVCache

    rng = np.random.default_rng(seed)
    g = lambda *s: _dev(rng.standard_normal(s).astype(np.float16))  # noqa: E731
    return dict(
        cache=KVCache.empty(64, heads, d, page), tables=torch.full((b, 12), -1, dtype=torch.int32, device="cuda"),
        held=torch.zeros(b, dtype=torch.int32, device="cuda"), free=torch.arange(64, dtype=torch.int32, device="cuda"),
        count=torch.tensor([64], dtype=torch.int32, device="cuda"), make=g, heads=heads, group=group, d=d, b=b)


def _one_step(st, added, q, k, v, n, most):
    from decode_kernel import append_kv, attend_kv, plan_kv_step

    step = plan_kv_step(st["tables"], st["held"], added, st["free"], st["count"], st["cache"].page_size, n)
    append_kv(st["cache"], k, v, step.slots)
    o = attend_kv(q, st["cache"], st["tables"], step.seq_lens, step.query_offsets, most)
    st["held"].copy_(step.seq_lens)
    st["count"].copy_(step.free_count)
    return o


def test_steps_follow_on():
    # Prompts, then tokens one by one, against attention over what read_kv
    # says the cache holds.
    st = _step_state(1)
    total = np.zeros(st["b"], int)
    for i, added in enumerate([[17, 0, 40, 1, 33], [1, 25, 1, 1, 1], [1] * 5, [0, 1, 0, 1, 1], [3, 2, 1, 0, 4]]):
        n = sum(added)
        q, k, v = (st["make"](n, st["heads"] * (st["group"] if j == 0 else 1), st["d"]) for j in range(3))
        o = _one_step(st, torch.tensor(added, dtype=torch.int32, device="cuda"), q, k, v, n, max(added))
        total += added
        assert st["held"].tolist() == total.tolist()
        host = _back(st["cache"])
        offs = np.concatenate([[0], np.cumsum(added)])
        ref, spread = kv_oracle.attend(q.float().cpu().numpy(), *host, st["tables"].cpu().numpy(), total, offs, st["d"]**-0.5, True)
        _check(o, ref, spread, total.max(), 127 * host[3].max(), torch.float16, f"step {i}")
    assert st["count"].tolist() == [64 - int(sum(-(-t // 16) for t in total))]


def test_graph_replays_match_eager():
    # A captured step, replayed with new inputs and lengths, against eager
    # steps on a twin; eager calls of other sizes between the replays.
    st, twin, other = _step_state(2), _step_state(2), _step_state(3, b=3, heads=1, group=9, d=64, page=32)
    b = st["b"]
    bufs = [st["make"](b, st["heads"] * (st["group"] if j == 0 else 1), st["d"]) for j in range(3)]
    added = torch.ones(b, dtype=torch.int32, device="cuda")
    for s in (st, twin):  # warm up: one step each
        _one_step(s, added, *bufs, b, 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _one_step(st, added, *bufs, b, 1)
    for i in range(40):
        for t in bufs:
            t.copy_(twin["make"](*t.shape))
        added.copy_(torch.tensor([(i + j) % 3 != 0 for j in range(b)], dtype=torch.int32))
        graph.replay()
        want = _one_step(twin, added, *bufs, b, 1)
        n = 21
        _one_step(other, torch.tensor([7, 7, 7], dtype=torch.int32, device="cuda"),
                  *(other["make"](n, 9 if j == 0 else 1, 64) for j in range(3)), n, 7)
        other["held"].zero_()
        other["count"].fill_(64)
        torch.cuda.synchronize()
        live = int(added.sum())
        assert torch.equal(out[:live], want[:live]), i
        assert torch.equal(st["held"], twin["held"]) and torch.equal(st["tables"], twin["tables"])


def test_on_another_stream():
    a, b = _step_state(4), _step_state(4)
    n = 31
    added = torch.tensor([31, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
    args = [a["make"](n, a["heads"] * (a["group"] if j == 0 else 1), a["d"]) for j in range(3)]
    want = _one_step(a, added, *args, n, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _one_step(b, added, *args, n, n)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_same_bits_again():
    rng = np.random.default_rng(10)
    from decode_kernel import attend_kv

    lens = [3000, 1, 700, 64]
    tables, pages = _tables(rng, lens, 16)
    cache = _cache(*_random_cache(rng, pages, 16, 4, 128))
    for new in ([1, 1, 1, 1], [300, 1, 200, 64]):
        offs = _dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
        q = _dev(rng.standard_normal((sum(new), 16, 128)).astype(np.float16))
        args = (q, cache, _dev(tables), _dev(np.array(lens, np.int32)), offs, max(new))
        first = attend_kv(*args)
        for _ in range(5):
            assert torch.equal(attend_kv(*args), first)


# ------------------------------------------------------------------- refusals
def test_refusals():
    from decode_kernel import KVCache, append_kv, attend_kv, plan_kv_step, read_kv

    cache = KVCache.empty(4, 2, 64, 16)
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    tables, slots = i32(0, 1)[None], torch.zeros(1, dtype=torch.int64, device="cuda")

    def bad(msg, fn, *args, **kw):
        with pytest.raises((RuntimeError, ValueError), match=msg):
            fn(*args, **kw)

    bad("head_size=96", KVCache.empty, 4, 2, 96)
    bad("page_size=48", KVCache.empty, 4, 2, 64, 48)
    bad("fp16 or bf16", append_kv, cache, k.float(), k.float(), slots)
    bad("one type", append_kv, cache, k, k.bfloat16(), slots)
    bad(r"\[tokens, 2, 64\]", append_kv, cache, k[:, :1], k[:, :1], slots)
    bad("int64", append_kv, cache, k, k, slots.int())
    bad("int64", append_kv, cache, k, k, torch.zeros(2, dtype=torch.int64, device="cuda"))
    bad("same device", append_kv, cache, k, k, slots.cpu())
    bad("cache's device", append_kv, cache, k.cpu(), k.cpu(), slots)
    bad("dtype", read_kv, cache, slots, torch.float64)
    bad("multiple of the cache's", attend_kv, q[:, :3], cache, tables, i32(1))
    bad("fp16 or bf16", attend_kv, q.float(), cache, tables, i32(1))
    bad("q_heads, 64", attend_kv, q[..., :32], cache, tables, i32(1))
    bad("seq_lens", attend_kv, q, cache, tables, i32(1, 2))
    bad("seq_lens", attend_kv, q, cache, tables, i32(1).long())
    bad("query_offsets", attend_kv, q, cache, tables, i32(1), i32(0, 1, 2))
    bad("one query", attend_kv, torch.cat([q, q]), cache, tables, i32(1))
    bad("max_query_len", attend_kv, q, cache, tables, i32(1), i32(0, 1), 0)
    bad("block_tables", attend_kv, q, cache, tables.long(), i32(1))
    bad("block_tables", attend_kv, q, cache, i32(0, 1, 2, 3).view(2, 2).t(), i32(1, 1))
    odd = KVCache(cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales[:3])
    bad("k_scales and v_scales", attend_kv, q, odd, tables, i32(1))
    odd = KVCache(cache.k_codes.transpose(0, 1), cache.v_codes.transpose(0, 1), cache.k_scales.t(), cache.v_scales.t())
    bad("contiguous", attend_kv, q, odd, tables, i32(1))
    odd = KVCache(cache.k_codes.float(), cache.v_codes, cache.k_scales, cache.v_scales)
    bad("int8", attend_kv, q, odd, tables, i32(1))
    bad("page_size", plan_kv_step, tables, i32(0), i32(1), i32(0), i32(1), 24, 1)
    bad("held", plan_kv_step, tables, i32(0, 0), i32(1), i32(0), i32(1), 16, 1)
    bad("free_count", plan_kv_step, tables, i32(0), i32(1), i32(0), i32(1, 1), 16, 1)
    bad("num_tokens", plan_kv_step, tables, i32(0), i32(1), i32(0), i32(1), 16, -1)
    many = torch.zeros(4097, dtype=torch.int32, device="cuda")
    bad("4096", plan_kv_step, many[:, None].contiguous(), many, many, i32(0), i32(1), 16, 1)


def test_nothing_to_do():
    from decode_kernel import KVCache, append_kv, attend_kv, read_kv

    cache = KVCache.empty(4, 2, 64, 16)
    none = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    no_slots = torch.zeros(0, dtype=torch.int64, device="cuda")
    append_kv(cache, none, none, no_slots)
    assert read_kv(cache, no_slots)[0].shape == (0, 2, 64)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    assert attend_kv(none, cache, i32().view(0, 3), i32()).shape == (0, 2, 64)
    q = torch.ones(2, 2, 64, dtype=torch.float16, device="cuda")
    # A table without columns and a cache without pages hold nothing: zeros.
    assert not attend_kv(q, cache, i32().view(2, 0), i32(5, 5)).any()
    empty = KVCache.empty(0, 2, 64, 16)
    assert not attend_kv(q, empty, i32(0, 1).view(2, 1), i32(5, 5)).any()
    append_kv(empty, q, q, torch.tensor([0, 1], device="cuda"))
    assert not read_kv(empty, torch.tensor([0, 1], device="cuda"))[1].any()
