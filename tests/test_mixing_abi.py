"""CPU checks of the C ABI of the gated delta rule, the short convolution and
the rotary positions (include/decode_kernel/dk_delta.h, dk_rotary.h): what is
refused, on the host and before any launch, and what is taken as nothing to do.
No call here reaches a GPU. The oracle's own checks, too."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from decode_kernel import _abi
from oracle import mixing_oracle

FAKE = 0x10000  # aligned, never dereferenced


@pytest.fixture(scope="module")
def lib():
    if not _abi.LIB_PATH.exists():
        pytest.fail(f"{_abi.LIB_PATH} is not built (python decode-kernel_amd/build_ext.py)")
    return _abi.load()


def _refused(lib, rc, text, status=_abi.DK_ERR_INVALID_ARGUMENT):
    assert rc == status, lib.dk_last_error().decode()
    assert text in lib.dk_last_error().decode()


def _delta(lib, out=FAKE, ws=FAKE, ws_bytes=1 << 40, **kw):
    f = dict(q=FAKE, k=FAKE, v=FAKE, log_decay=FAKE, beta=FAKE, states=FAKE, held=FAKE, offsets=FAKE, dtype=0, num_tokens=99,
             requests=2, qk_heads=2, v_heads=4, key_size=64, value_size=128, max_query_len=90, normalize=1, scale=1.0,
             **{f"{x}_{of}_stride": 512 for x in "qkv" for of in ("token", "head")})
    f.update(kw)
    return lib.dk_delta_rule(ctypes.byref(_abi.DeltaArgs(**f)), out, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "fp16 or bf16"), (dict(num_tokens=-1), ">= 0"), (dict(requests=-1), ">= 0"), (dict(requests=65536), "at most 65535"),
    (dict(qk_heads=0), "multiple"), (dict(qk_heads=3), "multiple"), (dict(v_heads=0), "multiple"), (dict(v_heads=65536), "multiple"),
    (dict(key_size=96), "64 or 128"), (dict(value_size=32), "64 or 128"), (dict(max_query_len=0), "max_query_len"),
    (dict(offsets=None), "one token"), (dict(q=None), "NULL"), (dict(beta=None), "NULL"), (dict(states=None), "NULL"),
    (dict(out=None), "NULL"), (dict(q=FAKE + 8), "16-byte"), (dict(states=FAKE + 4), "16-byte"), (dict(out=FAKE + 2), "16-byte"),
    (dict(log_decay=FAKE + 2), "4-byte"), (dict(offsets=FAKE + 1), "4-byte"), (dict(v_head_stride=100), "multiples of 8"),
    (dict(v_token_stride=2**24 + 8), "token strides"), (dict(q_token_stride=-8), "token strides"),
    (dict(ws=None), "workspace"), (dict(ws=FAKE + 128), "workspace"), (dict(ws_bytes=4096), "workspace"),
])
def test_delta_refuses(lib, kw, text):
    _refused(lib, _delta(lib, **kw), text)


def test_delta_refuses_what_no_index_holds(lib):
    _refused(lib, _delta(lib, num_tokens=2**31 - 1, v_heads=65534, qk_heads=2), "too large", _abi.DK_ERR_UNSUPPORTED)


def test_delta_without_args(lib):
    _refused(lib, lib.dk_delta_rule(None, FAKE, FAKE, 0, None), "NULL")


def test_delta_nothing_to_do(lib):
    assert _delta(lib, num_tokens=0, q=None, k=None, v=None, states=None, out=None, ws=None, ws_bytes=0) == _abi.DK_OK


def test_delta_workspace(lib):
    size = lib.dk_delta_workspace_bytes
    assert size(1000, 3, 2, 4, 128, 1) == 0  # tokens one by one need none
    assert size(0, 3, 2, 4, 128, 999) == size(1000, 3, 3, 4, 128, 999) == size(1000, 3, 2, 4, 96, 999) == 0
    one, two = size(1000, 3, 2, 4, 128, 999), size(2000, 3, 2, 4, 128, 999)
    assert 0 < one < two and one % 256 == 0


def test_more_than_a_launch_takes(lib):
    """A launch has fewer than 2^32 threads along x, and a call whose second launch
    would have more has changed the states in its first: refused before any."""
    _refused(lib, _delta(lib, num_tokens=64 * (2**22 - 2), max_query_len=2**28), "too large", _abi.DK_ERR_UNSUPPORTED)
    _refused(lib, _conv(lib, tokens=2**24, requests=2**24, offsets=None, channels=8), "too many", _abi.DK_ERR_UNSUPPORTED)
    _refused(lib, _conv(lib, tokens=8 * (2**24 - 3), channels=8), "too many", _abi.DK_ERR_UNSUPPORTED)
    _refused(lib, _rotate(lib, tokens=2**26 - 3, qh=1, kh=0, k=None, k_out=None), "too many", _abi.DK_ERR_UNSUPPORTED)
    _refused(lib, _rotate(lib, tokens=2**26 - 3, qh=64, kh=8), "too many", _abi.DK_ERR_UNSUPPORTED)


def test_delta_workspace_goes_by_requests_in_chunks(lib):
    """Requests of up to 16 tokens have no chunk: 3071 tokens can be those of 180
    others at most, whatever the batch's places are."""
    size = lib.dk_delta_workspace_bytes
    assert size(3071, 1024, 16, 32, 128, 2048) == size(3071, 180, 16, 32, 128, 2048) > size(3071, 179, 16, 32, 128, 2048)
    assert size(2048, 1, 16, 32, 128, 2048) < size(2048, 2, 16, 32, 128, 2048)


def _conv(lib, x=FAKE, stride=16, weight=FAKE, bias=None, windows=FAKE, held=None, offsets=FAKE, dtype=0, tokens=9, requests=2,
          channels=16, width=4, most=9, silu=1, y=FAKE):
    return lib.dk_short_conv(x, stride, weight, bias, windows, held, offsets, dtype, tokens, requests, channels, width, most,
                             silu, y, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "fp16 or bf16"), (dict(tokens=-1), ">= 0"), (dict(requests=-1), ">= 0"), (dict(channels=-1), ">= 0"),
    (dict(width=1), "width=1"), (dict(width=5), "width=5"), (dict(most=0), "max_query_len"), (dict(offsets=None), "one token"),
    (dict(x=None), "NULL"), (dict(weight=None), "NULL"), (dict(windows=None), "NULL"), (dict(y=None), "NULL"),
    (dict(x=FAKE + 1), "aligned"), (dict(bias=FAKE + 1), "aligned"), (dict(held=FAKE + 2), "aligned"),
])
def test_conv_refuses(lib, kw, text):
    _refused(lib, _conv(lib, **kw), text)


def test_conv_too_large_and_nothing_to_do(lib):
    _refused(lib, _conv(lib, channels=2**30 + 1), "too many", _abi.DK_ERR_UNSUPPORTED)
    assert _conv(lib, tokens=0, x=None, y=None, windows=None) == _conv(lib, channels=0, x=None) == _abi.DK_OK


def _rotate(lib, q=FAKE, qh=4, k=FAKE, kh=2, dtype=0, head_size=64, tokens=5, positions=FAKE, p64=0, axes=1, frequencies=FAKE,
            axis=None, count=32, q_out=FAKE, k_out=FAKE):
    return lib.dk_rotate_qk(q, 256, 64, qh, k, 128, 64, kh, dtype, head_size, tokens, positions, p64, axes, frequencies, axis,
                            count, 0, 0, q_out, k_out, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=2), "fp16 or bf16"), (dict(tokens=-1), ">= 0"), (dict(qh=-1), "heads"), (dict(kh=65536), "heads"),
    (dict(head_size=0), "head_size=0"), (dict(head_size=1025), "head_size=1025"), (dict(count=33), "num_frequencies=33"),
    (dict(head_size=1024, count=257), "num_frequencies=257"), (dict(count=-1), "num_frequencies=-1"), (dict(axes=0), "num_axes"),
    (dict(q=None), "NULL"), (dict(k_out=None), "NULL"), (dict(positions=None), "NULL"), (dict(frequencies=None), "NULL"),
    (dict(q=FAKE + 1), "aligned"), (dict(positions=FAKE + 4, p64=1), "aligned"), (dict(axis=FAKE + 2), "aligned"),
])
def test_rotate_refuses(lib, kw, text):
    _refused(lib, _rotate(lib, **kw), text)


def test_rotate_nothing_to_do(lib):
    assert _rotate(lib, tokens=0, q=None, positions=None) == _rotate(lib, qh=0, kh=0, q=None, k=None) == _abi.DK_OK


# ------------------------------------------------------------------ the oracle


def test_oracle_delta_by_hand():
    """One head of one column: numbers that can be followed."""
    q = k = np.array([[[3.0, 4.0]], [[4.0, -3.0]]])
    v, g, beta = np.array([[[10.0]], [[2.0]]]), np.log([[0.5], [0.25]]), np.array([[0.5], [1.0]])
    s = np.array([[[[1.0], [2.0]]]])
    out, after, reach = mixing_oracle.delta_rule(q, k, v, g, beta, s, offsets=[0, 2], scale=1.0, normalize=False)
    # 0.5 S = (0.5, 1); S^T k = 5.5; u = 0.5 * 4.5 = 2.25; S = (7.25, 10); S^T q = 61.75.
    # 0.25 S = (1.8125, 2.5); S^T k = -0.25; u = 2.25; S = (10.8125, -4.25); S^T q = 56.
    assert out.ravel().tolist() == [61.75, 56.0]
    assert after.ravel().tolist() == [10.8125, -4.25]
    assert np.allclose(reach.ravel() ** 2, [25 * (7.25**2 + 100), 25 * (10.8125**2 + 4.25**2)])


def test_oracle_conv_by_hand():
    x, w = np.array([[1.0], [2.0], [3.0]]), np.array([[10.0, 1.0]])
    y, after = mixing_oracle.short_conv(x, w, np.array([[[5.0]]]), offsets=[0, 3], silu=False)
    assert y.ravel().tolist() == [51.0, 12.0, 23.0] and after.ravel().tolist() == [3.0]
    y, _ = mixing_oracle.short_conv(x, w, np.array([[[5.0]]]), held=[0], offsets=[0, 3], bias=np.array([2.0]), silu=False)
    assert y.ravel().tolist() == [3.0, 14.0, 25.0]


def test_oracle_rotate_by_hand():
    x = np.array([[[1.0, 0.0, 0.0, 2.0, 9.0]]])
    got = mixing_oracle.rotate(x, [1], [np.pi / 2, np.pi])
    assert np.allclose(got, [[[0, 0, 1, -2, 9]]])
    got = mixing_oracle.rotate(x, [1], [np.pi / 2, np.pi], adjacent=True)
    assert np.allclose(got, [[[0, 1, 0, -2, 9]]])
    assert np.allclose(mixing_oracle.rotate(got, [1], [np.pi / 2, np.pi], adjacent=True, inverse=True), x)
