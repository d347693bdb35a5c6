"""short_conv and rotate_qk against their definitions in float64.

Tolerances. short_conv: a sum of up to 4 products and a bias in fp32 (each
operation 2^-24 of the terms' sum of magnitudes, 8 of them at most, and the
division and exponential of SiLU as many again, with a slope of at most 1.1), then
one rounding to the result's type. rotate_qk: cos and sin are within 2^-22 (the
turn's part rounded to fp32, times 2 pi, and the function's own last bits), two
products and a sum more, then one rounding.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from decode_kernel import Rotary, rotate_qk, short_conv
from oracle import mixing_oracle

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def f64(x):
    return None if x is None else x.double().cpu().numpy()


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------- short_conv


def conv_case(lens, channels, width, dtype=F16, bias=True, seed=0, lead=0, tail=0, held=None):
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()  # noqa: E731
    T = lead + sum(lens) + tail
    return dict(x=rand(T, channels), weight=rand(channels, width), windows=rand(len(lens), width - 1, channels),
                bias=rand(channels) if bias else None, held=[3 * (b % 2) for b in range(len(lens))] if held is None else held,
                offsets=[lead + int(n) for n in np.cumsum([0] + list(lens))])


def conv_run(c, most=None, silu=True):
    windows = c["windows"].clone()
    y = short_conv(c["x"], c["weight"], windows, None if c["held"] is None else ints(*c["held"]),
                   None if c["offsets"] is None else ints(*c["offsets"]), most, bias=c["bias"], silu=silu)
    return y, windows


def conv_check(c, most=None, silu=True):
    y, windows = conv_run(c, most, silu)
    want, kept = mixing_oracle.short_conv(f64(c["x"]), f64(c["weight"]), f64(c["windows"]), c["held"], c["offsets"],
                                          f64(c["bias"]), silu)
    terms, _ = mixing_oracle.short_conv(np.abs(f64(c["x"])), np.abs(f64(c["weight"])), np.abs(f64(c["windows"])), c["held"],
                                        c["offsets"], None if c["bias"] is None else np.abs(f64(c["bias"])), False)
    err = np.abs(f64(y) - want)
    bound = half_step(y.dtype) * np.abs(want) + 16 * 2.0**-24 * terms + 2.0**-25
    assert (err <= bound).all(), float((err / bound).max())
    assert np.array_equal(f64(windows), kept)  # inputs, not computed
    return y, windows


@pytest.mark.parametrize("channels", [1, 7, 8, 264, 2056])
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_conv_one_token_each(channels, width, dtype):
    c = conv_case([1] * 5, channels, width, dtype, seed=width)
    c["offsets"] = None
    conv_check(c)


@pytest.mark.parametrize("channels", [5, 64, 520])
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_conv_ragged(channels, width, dtype):
    lens = [1, 0, 2, 3, 15, 16, 17, 0, 4, 33, 100]
    conv_check(conv_case(lens, channels, width, dtype, seed=1, lead=2, tail=40))
    conv_check(conv_case(lens, channels, width, dtype, bias=False, seed=2), silu=False)


def test_conv_hundreds_of_requests():
    """Offsets are looked through 64 at a time."""
    lens = [(0, 1, 3, 17, 0, 2)[b % 6] for b in range(200)]
    for b in (0, 62, 63, 64, 65, 127, 128, 191, 192, 199):
        lens[b] = 30
    conv_check(conv_case(lens, 40, 4, seed=12, lead=1, tail=3))
    conv_check(conv_case(lens, 40, 4, seed=13), most=4)


def test_conv_many_tokens():
    """Where the chip is full anyway a workgroup takes 8 tokens."""
    conv_check(conv_case([5000, 1, 3200], 264, 4, BF16, seed=14, tail=5))


@pytest.mark.parametrize("most", [1, 4, 5, 16, 300])
def test_conv_max_query_len_only_picks_kernels(most):
    conv_check(conv_case([1, 40, 3, 4, 5], 72, 4, seed=3), most)


def test_conv_without_held_all_go_on():
    c = conv_case([5, 1], 16, 4, seed=4)
    c["held"] = None
    conv_check(c)


def test_conv_steps_are_one_step():
    c = conv_case([50], 24, 4, seed=5, held=[0])
    want, _ = conv_run(c)
    windows, got, at = torch.randn_like(c["windows"]), [], 0
    for n in (1, 1, 1, 20, 2, 25):
        got.append(short_conv(c["x"][at : at + n], c["weight"], windows, ints(at), ints(0, n), bias=c["bias"]))
        at += n
    assert torch.equal(torch.cat(got), want)
    assert torch.equal(windows[0], c["x"][-3:])


def test_conv_rows_of_nobody_and_bad_offsets():
    c = conv_case([20, 0, 2], 40, 3, seed=6, lead=20, tail=300)
    y, windows = conv_run(c)
    assert not y[:20].any() and not y[42:].any() and torch.equal(windows[1], c["windows"][1])
    for offsets in ([0, 30, 20, 40], [-1, 5, 10, 40], [0, 10, 20, 400]):
        c["offsets"] = offsets
        y, windows = conv_run(c)
        assert not y.any() and torch.equal(windows, c["windows"])
    c = conv_case([], 40, 3, seed=6, tail=33)
    y, _ = conv_run(c)
    assert y.shape == (33, 40) and not y.any()


def test_conv_not_finite_and_large():
    c = conv_case([30, 30], 16, 4, BF16, seed=7, held=[1, 1])
    clean, _ = conv_run(c)
    c["x"][35, 2] = float("nan")
    y, windows = conv_run(c)
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[35:39, 2] = False
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[35:39, 2]).all()
    # SiLU far out: 0 on the left, the value itself on the right.
    x = torch.tensor([-1e4, -200.0, 200.0, 3e4], dtype=BF16, device="cuda")[None].repeat(2, 1)
    w = torch.tensor([[0.0, 1.0]] * 4, dtype=BF16, device="cuda")
    y = short_conv(x, w, torch.zeros(2, 1, 4, dtype=BF16, device="cuda"))
    assert torch.equal(y[0, 2:], x[0, 2:]) and not y[0, :2].any()


def test_conv_strides_and_alignment():
    c = conv_case([9, 40], 64, 4, seed=8)
    want = conv_run(c)
    for pad in (8, 3):
        rows = torch.zeros(49, 64 + pad, dtype=F16, device="cuda")[:, pad:]
        rows.copy_(c["x"])
        got = conv_run({**c, "x": rows})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = conv_run({**c, "x": c["x"].t().contiguous().t()})
    assert torch.equal(got[0], want[0])
    weight = torch.zeros(64 * 4 + 1, dtype=F16, device="cuda")[1:].view(64, 4)
    weight.copy_(c["weight"])
    got = conv_run({**c, "weight": weight})
    assert torch.equal(got[0], want[0])


def test_conv_graph():
    c = conv_case([4, 20], 64, 4, seed=9)
    d = conv_case([4, 20], 64, 4, seed=10)
    want = [conv_run(x) for x in (c, d)]
    x, windows, offsets, held = c["x"].clone(), c["windows"].clone(), ints(*c["offsets"]), ints(*c["held"])
    call = lambda: short_conv(x, c["weight"], windows, held, offsets, 20, bias=c["bias"])  # noqa: E731
    d["weight"], d["bias"] = c["weight"], c["bias"]
    want = [conv_run(x) for x in (c, d)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for e, (wy, ww) in list(zip((c, d), want)) * 2:
        x.copy_(e["x"])
        windows.copy_(e["windows"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, wy) and torch.equal(windows, ww)
        conv_run(d)


def test_conv_refusals():
    c = conv_case([1, 1], 16, 4, seed=11)
    def call(x=c["x"], weight=c["weight"], windows=c["windows"], held=None, offsets=None, most=None, bias=None):
        return short_conv(x, weight, windows, held, offsets, most, bias=bias)
    for kw, text in [
        (dict(x=c["x"].float()), "fp16 or bf16"), (dict(weight=c["weight"].float()), "x's type"),
        (dict(weight=c["weight"][:8]), "weight"), (dict(weight=c["weight"][:, :1]), "width=1"),
        (dict(weight=torch.zeros(16, 5, device="cuda").half()), "width=5"), (dict(windows=c["windows"][:, :2]), "windows"),
        (dict(windows=c["windows"][:1]), "one token"), (dict(bias=c["weight"][:, 0]), "bias"),
        (dict(held=ints(1)), "held"), (dict(offsets=ints(0, 2)), "query_offsets"), (dict(most=0), "max_query_len"),
        (dict(x=c["x"].cpu()), "CUDA"), (dict(weight=c["weight"].cpu()), "device"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)


# ----------------------------------------------------------------- rotate_qk


def rotate_check(q, k, positions, rotary, inverse=False):
    got = rotate_qk(q, k, positions, rotary, inverse=inverse)
    for x, y in zip((q, k), got):
        want = mixing_oracle.rotate(f64(x), positions.cpu().numpy(), f64(rotary.frequencies),
                                    None if rotary.axes is None else rotary.axes.tolist(), rotary.adjacent, inverse)
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
        n = 2 * rotary.frequencies.numel()
        assert torch.equal(y[..., n:], x[..., n:])
        # A pair's length bounds what its cos and sin are multiplied by.
        a = f64(x[..., :n])
        other = (np.stack([a[..., 1::2], a[..., 0::2]], -1).reshape(a.shape) if rotary.adjacent
                 else np.concatenate([a[..., n // 2 :], a[..., : n // 2]], -1))
        err = np.abs(f64(y)[..., :n] - want[..., :n])
        bound = half_step(x.dtype) * np.abs(want[..., :n]) + (2.0**-21 + 2.0**-22) * (np.abs(a) + np.abs(other)) + 2.0**-25
        assert (err <= bound).all(), float((err / bound).max())
    return got


def heads_of(T, hq, hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(T, h, D, generator=g).to(dtype).cuda() for h in (hq, hk))


@pytest.mark.parametrize("D,R", [(128, 128), (128, 64), (64, 64), (80, 80), (32, 16), (256, 256), (96, 40), (10, 6), (7, 4), (2, 2), (6, 0)])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rotate_sizes(D, R, adjacent, dtype):
    q, k = heads_of(19, 6, 2, D, dtype, seed=D)
    f = (10000.0 ** (-torch.arange(R // 2).double() * 2 / max(R, 1))).float().cuda()
    positions = torch.randint(0, 5000, (19,), generator=torch.Generator().manual_seed(1)).int().cuda()
    rotate_check(q, k, positions, Rotary(f, None, adjacent))
    rotate_check(q, k, positions.long(), Rotary(f, None, adjacent), inverse=True)


@pytest.mark.parametrize("T", [1, 2, 3, 5, 64, 700])
@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 1), (64, 8), (5, 0), (0, 3)])
def test_rotate_counts(T, hq, hk):
    q, k = heads_of(T, hq, hk, 128, BF16, seed=T)
    rotate_check(q, k, torch.arange(T, device="cuda").int(), Rotary.from_base(128))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [(16, 24, 24), (22, 21, 21), (64, 0), (0, 32, 32), (1, 1, 1, 61)])
def test_rotate_axes(interleaved, sections):
    rotary = Rotary.from_base(128, sections=sections, interleaved=interleaved)
    if not interleaved:
        assert [rotary.axes.tolist().count(a) for a in range(len(sections))] == list(sections)
    q, k = heads_of(33, 4, 2, 128, F16, seed=3)
    positions = torch.randint(0, 900, (len(sections), 33), generator=torch.Generator().manual_seed(2)).cuda()
    rotate_check(q, k, positions, rotary)
    rotate_check(q, k, positions.int(), rotary, inverse=True)


def test_interleaved_sections_share_out_every_speed():
    axes = Rotary.from_base(128, sections=(24, 20, 20), interleaved=True).axes.tolist()
    assert axes[:6] == [0, 1, 2, 0, 1, 2] and axes[60:] == [0] * 4
    assert [axes.count(a) for a in range(3)] == [24, 20, 20]


def test_far_positions_are_exact():
    q, k = heads_of(6, 2, 1, 64, F16, seed=4)
    far = torch.tensor([0, 1, 131071, 10**6 + 1, 2**31 - 1, -7], device="cuda")
    rotate_check(q, k, far, Rotary.from_base(64))
    rotate_check(q, k, far.int(), Rotary.from_base(64))
    rotate_check(q, k, far * 1000 + 3, Rotary.from_base(64, base=1e6))


def test_axes_outside_are_the_nearest():
    q, k = heads_of(5, 1, 1, 16, F16, seed=5)
    positions = torch.arange(10, device="cuda").int().view(2, 5)
    f = torch.rand(8, generator=torch.Generator().manual_seed(3)).cuda()
    rotate_check(q, k, positions, Rotary(f, ints(-3, 0, 1, 2, 9, 1, 0, 1)))


def test_inverse_is_the_gradient():
    """Against the formula's gradient by differences: y is linear in x, so a
    difference of two results is exact but for their roundings."""
    q, k = heads_of(4, 2, 1, 32, F16, seed=6)
    rotary, positions = Rotary.from_base(32), ints(3, 0, 77, 1000)
    gq, gk = heads_of(4, 2, 1, 32, F16, seed=7)
    back_q, back_k = rotate_qk(gq, gk, positions, rotary, inverse=True)
    for x, g, back, other in ((q, gq, back_q, k), (k, gk, back_k, q)):
        dot = lambda p: float((rotate_qk(p, other if p is q else other, positions, rotary)[0].double() * g.double()).sum())  # noqa: E731
        # <R x, g> = <x, R^T g>: both sides hold x's and g's values with one rounding each.
        n = x.numel()
        size = float((x.double().abs().amax() * g.double().abs().amax()))
        assert abs(dot(x) - float((x.double() * back.double()).sum())) <= 4 * half_step(F16) * size * n**0.5
        e = torch.zeros_like(x)
        e[2, 0, 5] = 1.0
        assert abs(dot(e) - float(back[2, 0, 5])) <= 4 * half_step(F16) * float(g.abs().amax()) + 2.0**-24
    again_q, again_k = rotate_qk(*rotate_qk(q, k, positions, rotary), positions, rotary, inverse=True)
    for x, y in ((q, again_q), (k, again_k)):
        # Two roundings of a pair, whose length the rotations keep.
        assert ((x.double() - y.double()).abs() <= 4 * half_step(F16) * x.double().abs().amax()).all()


@pytest.mark.parametrize("pad", [0, 8, 4, 1])
def test_rotate_slices(pad):
    """Slices of one projection, at rows and addresses that allow wide loads and that do not."""
    T = 21
    rows = torch.randn(T, 12 * 64 + pad, generator=torch.Generator().manual_seed(8)).half().cuda()[:, pad:]
    q, k, _ = rows.split([8 * 64, 2 * 64, 2 * 64], 1)
    q, k = q.unflatten(1, (8, 64)), k.unflatten(1, (2, 64))
    rotary, positions = Rotary.from_base(64), torch.arange(T, device="cuda")
    want = rotate_check(q.contiguous(), k.contiguous(), positions, rotary)
    for a, b in ((q, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(1, 2).contiguous().transpose(1, 2))):
        got = rotate_qk(a, b, positions, rotary)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rotate_empty_and_special():
    rotary = Rotary.from_base(64)
    q, k = heads_of(0, 4, 2, 64, F16)
    out = rotate_qk(q, k, torch.zeros(0, dtype=torch.int32, device="cuda"), rotary)
    assert out[0].shape == q.shape and out[1].shape == k.shape
    q, k = heads_of(3, 4, 2, 64, F16)
    clean = rotate_qk(q, k, ints(1, 2, 3), rotary)
    q[1, 2, 5] = float("nan")
    got = rotate_qk(q, k, ints(1, 2, 3), rotary)
    keep = torch.ones_like(q, dtype=torch.bool)
    keep[1, 2, [5, 37]] = False
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.isnan(got[0][1, 2, [5, 37]]).all()
    assert torch.equal(rotate_qk(q[:1], k[:1], ints(0), rotary)[0], q[:1])  # position 0 turns nothing


def test_rotate_graph_and_stream():
    rotary = Rotary.from_base(128, sections=(16, 24, 24))
    sets = [(*heads_of(9, 8, 2, 128, BF16, seed=s), torch.randint(0, 99, (3, 9), generator=torch.Generator().manual_seed(s)).cuda())
            for s in range(2)]
    want = [rotate_qk(*s, rotary) for s in sets]
    q, k, p = (x.clone() for x in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotate_qk(q, k, p, rotary)
    side.synchronize()
    assert torch.equal(got[0], want[0][0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oq, ok = rotate_qk(q, k, p, rotary)
    for s, (wq, wk) in list(zip(sets, want)) * 2:
        for x, y in zip((q, k, p), s):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(oq, wq) and torch.equal(ok, wk)
        rotate_qk(*sets[1], rotary)


def test_rotate_refusals():
    rotary = Rotary.from_base(64)
    q, k = heads_of(3, 4, 2, 64, F16)
    p = ints(0, 1, 2)
    for args, text in [
        ((q.float(), k.float(), p, rotary), "fp16 or bf16"), ((q, k.bfloat16(), p, rotary), "one type"),
        ((q, k[:2], p, rotary), "tokens, heads"), ((q, k, p[:2], rotary), "positions"), ((q, k, p.float(), rotary), "positions"),
        ((q, k, p.repeat(2, 1), rotary), "axis of each"), ((q, k, p, Rotary(rotary.frequencies.double())), "frequencies"),
        ((q, k, p, Rotary.from_base(66)), "frequencies"), ((q, k, p, Rotary(rotary.frequencies, ints(0))), "axes"),
        ((q.cpu(), k.cpu(), p, rotary), "CUDA"), ((q, k, p.cpu(), rotary), "device"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            rotate_qk(*args)
    for bad in (dict(rotary_size=63), dict(rotary_size=0), dict(rotary_size=64, sections=(1, 2)), dict(rotary_size=64, sections=(33, -1))):
        with pytest.raises(ValueError):
            Rotary.from_base(**bad)
