"""CPU checks of the key/value cache's C ABI (include/decode_kernel/dk_kv.h):
what it refuses, on the host and before any launch, and what it takes as
nothing to do. No call here reaches a GPU."""

from __future__ import annotations

import ctypes

import pytest

from decode_kernel import _abi

FAKE = 0x10000  # aligned, never dereferenced


@pytest.fixture(scope="module")
def lib():
    if not _abi.LIB_PATH.exists():
        pytest.fail(f"{_abi.LIB_PATH} is not built (python decode-kernel_amd/build_ext.py)")
    return _abi.load()


def _cache(**kw):
    f = dict(k_codes=FAKE, v_codes=FAKE, k_scales=FAKE, v_scales=FAKE, pages=4, heads=2, head_size=64, page_size=16)
    f.update(kw)
    return _abi.KvCache(**f)


def _refused(lib, rc, text, status=_abi.DK_ERR_INVALID_ARGUMENT):
    assert rc == status
    assert text in lib.dk_last_error().decode()


BAD_CACHES = [
    (dict(page_size=0), "page_size=0"), (dict(page_size=48), "page_size=48"), (dict(page_size=256), "page_size=256"),
    (dict(head_size=96), "head_size=96"), (dict(pages=-1), "pages >= 0"), (dict(heads=0), "heads"),
    (dict(heads=65536), "heads"), (dict(k_codes=None), "NULL"), (dict(v_scales=None), "NULL"),
    (dict(v_codes=FAKE + 8), "16-byte"), (dict(k_scales=FAKE + 2), "4-byte"),
]


def _attend(lib, cache, q=FAKE, dtype=0, qt=256, qh=64, tables=FAKE, width=3, lens=FAKE, offsets=FAKE, tokens=2,
            requests=2, q_heads=4, most=1, out=FAKE, ws=FAKE, ws_bytes=1 << 40):
    return lib.dk_kv_attend(q, dtype, qt, qh, ctypes.byref(cache) if cache else None, tables, width, lens, offsets,
                            tokens, requests, q_heads, most, 1.0, 1, out, ws, ws_bytes, None)


def _append(lib, cache, k=FAKE, v=FAKE, dtype=0, strides=(128, 64, 128, 64), slots=FAKE, tokens=2):
    return lib.dk_kv_append(ctypes.byref(cache) if cache else None, k, v, dtype, *strides, slots, tokens, None)


def _read(lib, cache, slots=FAKE, tokens=2, dtype=0, k=FAKE, v=FAKE):
    return lib.dk_kv_read(ctypes.byref(cache) if cache else None, slots, tokens, dtype, k, v, None)


@pytest.mark.parametrize("fields,text", BAD_CACHES)
def test_bad_caches(lib, fields, text):
    for call in (_attend, _append, _read):
        _refused(lib, call(lib, _cache(**fields)), text)


def test_no_cache(lib):
    for call in (_attend, _append, _read):
        _refused(lib, call(lib, None), "cache must not be NULL")


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "fp16 or bf16"), (dict(dtype=-1), "fp16 or bf16"), (dict(tokens=-1), ">= 0"), (dict(requests=-1), ">= 0"),
    (dict(width=-1), ">= 0"), (dict(q_heads=0), "multiple"), (dict(q_heads=3), "multiple"),
    (dict(offsets=None, tokens=3), "one query"), (dict(most=0), "max_query_len"), (dict(q=None), "NULL"),
    (dict(out=None), "NULL"), (dict(lens=None), "NULL"), (dict(tables=None), "NULL"), (dict(ws=None), "NULL"),
    (dict(q=FAKE + 8), "16-byte"), (dict(out=FAKE + 2), "16-byte"), (dict(ws=FAKE + 8), "16-byte"),
    (dict(qt=100), "multiples of 8"), (dict(qh=60), "multiples of 8"), (dict(ws_bytes=64), "workspace"),
    (dict(width=2**27), "fit in int32"),
])
def test_attend_refuses(lib, kw, text):
    _refused(lib, _attend(lib, _cache(), **kw), text)


def test_attend_refuses_what_no_index_holds(lib):
    rc = _attend(lib, _cache(heads=1), tokens=2**30, q_heads=4, most=9)
    _refused(lib, rc, "too large", _abi.DK_ERR_UNSUPPORTED)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "fp16 or bf16"), (dict(tokens=-1), ">= 0"), (dict(k=None), "NULL"), (dict(v=None), "NULL"),
    (dict(slots=None), "NULL"), (dict(k=FAKE + 8), "16-byte"), (dict(slots=FAKE + 4), "8-byte"),
    (dict(strides=(128, 64, 128, 60)), "multiples of 8"), (dict(strides=(4, 64, 128, 64)), "multiples of 8"),
])
def test_append_refuses(lib, kw, text):
    _refused(lib, _append(lib, _cache(), **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), "fp16, bf16 or fp32"), (dict(tokens=-1), ">= 0"), (dict(k=None), "NULL"), (dict(slots=None), "NULL"),
    (dict(v=FAKE + 8), "16-byte"), (dict(slots=FAKE + 4), "8-byte"),
])
def test_read_refuses(lib, kw, text):
    _refused(lib, _read(lib, _cache(), **kw), text)


def _plan(lib, tables=FAKE, width=4, held=FAKE, added=FAKE, requests=2, free=FAKE, capacity=9, count=FAKE, page=16,
          tokens=5, slots=FAKE, positions=FAKE, offsets=FAKE, lens=FAKE, count_out=FAKE + 16):
    return lib.dk_kv_plan(tables, width, held, added, requests, free, capacity, count, page, tokens, slots, positions,
                          offsets, lens, count_out, None)


@pytest.mark.parametrize("kw,text", [
    (dict(page=24), "page_size=24"), (dict(requests=-1), "requests"), (dict(requests=_abi.DK_KV_MAX_REQUESTS + 1), "4096"),
    (dict(width=-1), ">= 0"), (dict(tokens=-1), ">= 0"), (dict(capacity=-1), ">= 0"), (dict(width=2**28), "fit in int32"),
    (dict(tables=None), "NULL"), (dict(held=None), "NULL"), (dict(added=None), "NULL"), (dict(free=None), "NULL"),
    (dict(count=None), "NULL"), (dict(slots=None), "NULL"), (dict(positions=None), "NULL"), (dict(offsets=None), "NULL"),
    (dict(lens=None), "NULL"), (dict(count_out=None), "NULL"), (dict(count_out=FAKE), "must not be free_count"),
])
def test_plan_refuses(lib, kw, text):
    _refused(lib, _plan(lib, **kw), text)


def test_nothing_to_do(lib):
    assert _attend(lib, _cache(), q=None, tokens=0, requests=0) == _abi.DK_OK
    assert _append(lib, _cache(), k=None, tokens=0) == _abi.DK_OK
    assert _append(lib, _cache(pages=0, k_codes=None)) == _abi.DK_OK
    assert _read(lib, _cache(), k=None, tokens=0) == _abi.DK_OK


def test_workspace_bytes(lib):
    ws = lib.dk_kv_attend_workspace_bytes
    assert ws(0, 4, 8, 2, 128, 10, 16, 1) == 0 and ws(4, 0, 8, 2, 128, 10, 16, 1) == 0
    assert ws(4, 4, 8, 0, 128, 10, 16, 1) == 0
    # Bounded, whatever the lengths: a call's partial results, not its scores.
    for args in ((1, 1, 64, 8, 128, 2**20, 128, 1), (4096, 1, 64, 8, 128, 2**20, 16, 4096), (8192, 256, 32, 32, 64, 4096, 16, 8192)):
        assert 0 < ws(*args) <= 256 << 20, args
