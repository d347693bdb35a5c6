"""delta_rule, short_conv and rotate_qk together with the plan, the cache and
the 4-bit projections: examples/hybrid_decode.py a step at a time against one
step over the whole sequences, a captured decode step, and sizes past 32 bits."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from decode_kernel import delta_rule, plan_kv_step, rotate_qk, short_conv, Rotary

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "hybrid_decode.py"
PROMPTS = (37, 5, 0, 130, 64)


def _example():
    spec = importlib.util.spec_from_file_location("hybrid_decode", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _prompts():
    g = torch.Generator().manual_seed(2)
    return [torch.randint(0, 1000, (n,), generator=g).tolist() for n in PROMPTS]


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_steps_against_one_step():
    ex = _example()
    model, prompts = ex.Hybrid(), _prompts()
    out, last, batch = ex.generate(model, prompts, 20)
    want, whole = ex.again(model, prompts, out)
    live = [0, 1, 3, 4]
    # The cache's codes are off by half a step of 1/127 of a page's largest, once
    # more for each time its scale grew: about 1% of a value, which softmax and
    # sums average; the logits' own size is 1.
    err = (want[live] - last[live]).float()
    assert (err.norm() / want[live].float().norm()).item() < 0.05
    assert batch.held.tolist() == whole.held.tolist() == [57, 25, 0, 150, 84]
    # The first layer mixes before any attention: its inputs differ by the last
    # fp16 bit of its projection (2^-11 of a value; another number of rows may
    # take another kernel), its states by as much of their size and not more
    # where errors of q, k and v add: 4 * 2^-11.
    a, b = batch.memory[0]["states"][live], whole.memory[0]["states"][live]
    assert ((a - b).norm() / b.norm()).item() < 4 * 2.0**-11


def test_a_place_is_used_again():
    """Another request in places that held one, with nothing cleared between."""
    ex = _example()
    model, prompts = ex.Hybrid(2), _prompts()
    batch = ex.Batch(model, len(prompts), 200)
    want = ex.run_prompts(model, batch, prompts)
    batch.held.zero_()
    batch.tables.fill_(-1)
    batch.free_count.fill_(batch.free.numel())
    batch.free.copy_(torch.arange(batch.free.numel()).int())
    got = ex.run_prompts(model, batch, prompts)
    live = [0, 1, 3, 4]
    assert torch.equal(got[live], want[live])


def test_captured_decode_step():
    """One captured step replayed over the tokens, against the same steps run eagerly."""
    ex = _example()
    model, prompts = ex.Hybrid(), _prompts()
    torch.manual_seed(0)
    eager, captured = (ex.Batch(model, len(prompts), 200) for _ in range(2))
    for batch in (eager, captured):
        ex.run_prompts(model, batch, prompts)
    live, ids = ints(1, 1, 0, 1, 1), torch.tensor([1, 2, 3, 4], device="cuda")
    held, count = captured.held.clone(), captured.free_count.clone()
    tokens = ids.clone()

    def call():
        captured.held, captured.free_count = held, count
        logits, step = captured.run(model, tokens, live, 1)
        held.copy_(step.seq_lens)
        count.copy_(step.free_count)
        return logits

    keep = [x.clone() for m in captured.memory for x in (m.values() if isinstance(m, dict) else
            (m.k_codes, m.v_codes, m.k_scales, m.v_scales))] + [captured.tables.clone(), held.clone(), count.clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    now = [x for m in captured.memory for x in (m.values() if isinstance(m, dict) else
           (m.k_codes, m.v_codes, m.k_scales, m.v_scales))] + [captured.tables, held, count]
    for x, y in zip(now, keep):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = call()
    for i in range(6):
        want, _ = eager.run(model, ids + 7 * i, live, 1)
        tokens.copy_(ids + 7 * i)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want), i


def test_places_past_the_last_token():
    """A step of 64 places with 21 tokens of three requests: the other rows are zeros and nobody's state moves."""
    tables = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    held = ints(0, 4, 9)
    step = plan_kv_step(tables, held, ints(18, 0, 3), ints(*range(20)), ints(20), 16, 64)
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    states, windows = rand(3, 2, 64, 64), rand(3, 3, 256).half()
    before = states.clone(), windows.clone()
    rows = short_conv(rand(64, 256).half(), rand(256, 4).half(), windows, held, step.query_offsets, 18)
    q, k, v = (t.unflatten(1, (-1, 64)) for t in rows.split([64, 64, 128], 1))
    o = delta_rule(q, k, v, -rand(64, 2).abs(), rand(64, 2).sigmoid(), states, held, step.query_offsets, 18)
    assert not rows[21:].any() and not o[21:].any() and rows[:21].any() and o[:21].any()
    assert torch.equal(states[1], before[0][1]) and torch.equal(windows[1], before[1][1])
    assert not torch.equal(states[0], before[0][0]) and not torch.equal(windows[2], before[1][2])
    q2, k2 = rotate_qk(q, k, step.positions, Rotary.from_base(64))
    assert torch.isfinite(q2).all() and torch.isfinite(k2).all()


def test_states_past_32_bits():
    """4500 states of 32 heads: their elements pass 2^31. A request at either end against the same alone."""
    B, H = 4500, 32
    states = torch.zeros(B, H, 128, 128, device="cuda")
    assert states.numel() > 2**31
    g = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, v = rand(B, H, 128).half(), rand(B, H, 128).half(), rand(B, H, 128).half()
    decay, beta = -rand(B, H).abs(), rand(B, H).sigmoid()
    states[0], states[-1] = rand(H, 128, 128), rand(H, 128, 128)
    alone = [(states[b : b + 1].clone() if b >= 0 else states[-1:].clone()) for b in (0, -1)]
    o = delta_rule(q, k, v, decay, beta, states)
    for b, s in zip((0, B - 1), alone):
        at = slice(b, b + 1)
        assert torch.equal(delta_rule(q[at], k[at], v[at], decay[at], beta[at], s), o[at])
        assert torch.equal(s, states[at])


def test_rows_past_32_bits():
    """Rows of 2^31 elements and more: the last request, a prompt in chunks, against the same rows alone."""
    T, H = 280000, 64
    rows = torch.empty(T, H * 128, device="cuda", dtype=torch.float16)
    assert rows.numel() > 2**31
    rows.normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    x = rows.view(T, H, 128)
    g = torch.Generator(device="cuda").manual_seed(6)
    decay, beta = -torch.rand(T, 1, device="cuda", generator=g).expand(T, H).contiguous(), torch.full((T, H), 0.5, device="cuda")
    states = torch.zeros(2, H, 128, 128, device="cuda")
    last = T - 300
    offsets = ints(last, last + 20, T)  # the rows before are nobody's
    o = delta_rule(x, x, x, decay, beta, states, None, offsets, 280)
    small = torch.zeros(2, H, 128, 128, device="cuda")
    part = x[last:]
    want = delta_rule(part, part, part, decay[last:], beta[last:], small, None, ints(0, 20, 300), 280)
    assert torch.equal(o[last:], want) and torch.equal(states, small)
    assert not o[:last].any()
    y, w = torch.zeros(2, 3, H * 128, dtype=torch.float16, device="cuda"), torch.ones(H * 128, 4, dtype=torch.float16, device="cuda")
    del o
    c = short_conv(rows, w, y, None, offsets, 280)
    z = torch.zeros_like(y)
    assert torch.equal(c[last:], short_conv(rows[last:], w, z, None, ints(0, 20, 300), 280)) and torch.equal(y, z)
    del c
    rotary = Rotary.from_base(128)
    a, b = rotate_qk(x, x[:, :1], torch.arange(T, device="cuda"), rotary)
    a2, b2 = rotate_qk(part, part[:, :1], torch.arange(last, T, device="cuda"), rotary)
    assert torch.equal(a[last:], a2) and torch.equal(b[last:], b2)
