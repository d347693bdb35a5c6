"""delta_rule against the rule in float64, token by token.

Tolerances. The result is rounded once, by at most half a step of its type
(eps / 2 relative). Before that everything is fp32 (or fp32 in parts of 22
bits): with keys of length one and beta up to 1 a token's step does not enlarge
what stood in a column of the state, so a column's error is a few roundings of
2^-24 for each of the key_size terms of its sums, which add like a random walk,
and those that earlier tokens left, which fade. SUM = 8 sqrt(key_size) 2^-24 of
a column's size covers it (SUM twice for an output, whose own sum over the keys' axis rounds
as much again).
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from decode_kernel import delta_rule
from oracle import mixing_oracle

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def case(lens, heads=2, group=1, dk=64, dv=64, dtype=F16, seed=0, lead=0, tail=0, held=None):
    """Inputs of requests with `lens` new tokens each; rows of nobody before and after."""
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    B, T, Hv = len(lens), lead + sum(lens) + tail, heads * group
    c = dict(q=rand(T, heads, dk).to(dtype), k=rand(T, heads, dk).to(dtype), v=rand(T, Hv, dv).to(dtype),
             log_decay=-torch.rand(T, Hv, generator=g).pow(3) * 2, beta=torch.rand(T, Hv, generator=g),
             states=0.3 * rand(B, Hv, dk, dv))
    c = {n: x.cuda() for n, x in c.items()}
    c["offsets"] = [lead + int(x) for x in np.cumsum([0] + list(lens))]
    c["held"] = [5 * (b % 3) for b in range(B)] if held is None else held
    return c


def run(c, max_query_len=None, **kw):
    """The call, on clones of what it updates."""
    states = c["states"].clone()
    offsets = None if c["offsets"] is None else ints(*c["offsets"])
    held = None if c["held"] is None else ints(*c["held"])
    o = delta_rule(c["q"], c["k"], c["v"], c["log_decay"], c["beta"], states, held, offsets, max_query_len, **kw)
    return o, states


def expect(c, **kw):
    f = lambda x: x.double().cpu().numpy()  # noqa: E731
    return mixing_oracle.delta_rule(f(c["q"]), f(c["k"]), f(c["v"]), f(c["log_decay"]), f(c["beta"]), f(c["states"]),
                                    c["held"], c["offsets"], **kw)


def part(dk):
    return 8 * dk**0.5 * 2.0**-24


def close_states(got, want, dk):
    """Column by column: a column runs over the keys' axis."""
    x, y = got.double().cpu().numpy(), np.asarray(want)
    assert x.shape == y.shape and np.isfinite(x).all()
    bound = part(dk) * np.sqrt((y * y).sum(-2, keepdims=True)) + 2.0**-60
    err = np.abs(x - y)
    assert (err <= bound).all(), float((err / bound).max())


def close_out(got, want, reach, dk):
    """An output is scale q . column: where the column's error is at most SUM of
    its size, the output's is at most SUM scale |q| |column| = SUM reach, however
    small q . column itself came out. Then one rounding (of fp16 by 2^-25 where
    its step stays 2^-24)."""
    x, y = got.double().cpu().numpy(), np.asarray(want)
    assert x.shape == y.shape and np.isfinite(x).all()
    bound = torch.finfo(got.dtype).eps / 2 * np.abs(y) + 2 * part(dk) * reach
    bound += 2.0**-25 if got.dtype == F16 else 2.0**-60
    err = np.abs(x - y)
    assert (err <= bound).all(), float((err / bound).max())


def check(c, max_query_len=None, **kw):
    o, states = run(c, max_query_len, **kw)
    want_o, want_s, reach = expect(c, **kw)
    close_out(o, want_o, reach, c["q"].shape[-1])
    close_states(states, want_s, c["q"].shape[-1])
    return o, states


SHAPES = [(2, 1, 64, 64), (1, 3, 128, 64), (2, 2, 64, 128), (4, 1, 128, 128)]


@pytest.mark.parametrize("heads,group,dk,dv", SHAPES)
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("B", [1, 5])
def test_one_token_each(heads, group, dk, dv, dtype, B):
    c = case([1] * B, heads, group, dk, dv, dtype, seed=B)
    c["offsets"] = None
    check(c)


def test_without_held_all_go_on():
    c = case([1, 1, 1], seed=3)
    c["held"] = None
    check(c)
    c = case([70, 3], seed=4)
    c["held"] = None
    check(c)


@pytest.mark.parametrize("heads,group,dk,dv", SHAPES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_few_tokens(heads, group, dk, dv, dtype):
    check(case([4, 0, 2, 9, 1], heads, group, dk, dv, dtype, seed=1, lead=3, tail=2), max_query_len=9)


@pytest.mark.parametrize("heads,group,dk,dv", SHAPES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_prompts(heads, group, dk, dv, dtype):
    check(case([65, 0, 1, 200, 17, 64, 16, 63], heads, group, dk, dv, dtype, seed=2, lead=5, tail=70))


@pytest.mark.parametrize("n", [17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129])
@pytest.mark.parametrize("held", [0, 7])
def test_lengths_around_chunks(n, held):
    check(case([n], 2, 2, 128, 64, BF16, seed=n, held=[held]))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_long(dtype):
    check(case([1111], 1, 2, 128, 128, dtype, seed=5, held=[3]))


def test_max_query_len_only_picks_kernels():
    c = case([100, 3, 1], 2, 2, 64, 128, seed=6)
    for most in (1, 16, 17, 1000):
        check(c, max_query_len=most)


@pytest.mark.parametrize("most", [None, 17, 600, 10**6])
def test_more_prompts_than_seem_to_be(most):
    """One long prompt among many short ones: the workgroups are counted by the
    longest and take several prompts each."""
    lens = [600] + [20, 0, 3] * 12 + [65, 1, 129]
    check(case(lens, 1, 2, 64, 64, BF16, seed=33), max_query_len=most)


@pytest.mark.parametrize("most", [1, 70])
def test_hundreds_of_requests(most):
    """Offsets are looked through 64 at a time: long requests at either side of
    those borders, and empty ones."""
    lens = [(0, 1, 3, 17, 0, 2)[b % 6] for b in range(200)]
    for b in (0, 62, 63, 64, 65, 127, 128, 191, 192, 199):
        lens[b] = 70
    check(case(lens, 1, 1, 64, 64, seed=34, lead=1, tail=3), max_query_len=most)


def test_split_steps_are_one_step():
    """A prompt in two steps and then tokens one by one ends where one step does."""
    c = case([90], 2, 1, 128, 128, BF16, seed=7, held=[0])
    want_o, want_s, reach = expect(c)
    states = torch.randn_like(c["states"])  # what another request left
    got, at, held = [], 0, 0
    for n in (33, 50, 1, 1, 5):
        part = {x: c[x][at : at + n] for x in ("q", "k", "v", "log_decay", "beta")}
        got.append(delta_rule(**part, states=states, held=ints(held), query_offsets=ints(0, n)))
        at, held = at + n, held + n
    close_out(torch.cat(got), want_o, reach, 128)
    close_states(states, want_s, 128)


@pytest.mark.parametrize("n", [9, 90])
def test_scale_and_given_lengths(n):
    c = case([n], seed=8)
    c["k"] = torch.nn.functional.normalize(c["k"].float(), dim=-1).half()
    check(c, scale=0.7, normalize=False)


@pytest.mark.parametrize("n", [5, 150])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_of_any_size(n, dtype):
    """Keys, queries and values of lengths far apart, and zeros."""
    c = case([n], 2, 1, 128, 64, dtype, seed=9, held=[1])
    power = torch.randint(-6, 5, (n, 2, 1), generator=torch.Generator().manual_seed(1)).cuda()
    c["k"] = (c["k"].float() * 2.0**power).to(dtype)
    c["q"] = (c["q"].float() * 2.0 ** -power).to(dtype)
    c["k"][n // 2] = 0
    c["q"][n // 3] = 0
    c["v"][n // 4] = 0
    check(c)


@pytest.mark.parametrize("n", [5, 150])
def test_columns_of_any_size(n):
    """Values whose columns lie twelve powers of ten apart keep each its accuracy."""
    c = case([n], 1, 1, 64, 64, BF16, seed=10, held=[1])
    size = 10.0 ** torch.linspace(-6, 6, 64, device="cuda")
    c["v"], c["states"] = (c["v"].float() * size).to(BF16), c["states"] * size
    check(c)


@pytest.mark.parametrize("n", [6, 130])
@pytest.mark.parametrize("log_decay", [0.0, -1e-4, -1.0, -30.0, -200.0, -float("inf")])
def test_decays(n, log_decay):
    c = case([n], seed=11, held=[1])
    c["log_decay"].fill_(log_decay)
    check(c)


@pytest.mark.parametrize("n", [6, 130])
def test_decays_far_apart(n):
    """A state that is emptied now and then among decays of every size."""
    c = case([n], seed=12, held=[1])
    c["log_decay"][1::7] = -float("inf")
    c["log_decay"][2::7] = -90.0
    c["log_decay"][3::7] = 0.0
    check(c)


@pytest.mark.parametrize("n", [6, 130])
@pytest.mark.parametrize("beta", [0.0, 1.0])
def test_betas(n, beta):
    c = case([n], seed=13, held=[1])
    c["beta"].fill_(beta)
    check(c)


def one_key(beta):
    c = case([150], seed=14, held=[1])
    c["k"][:] = c["k"][:1].clone()
    c["beta"].fill_(beta)
    c["log_decay"].zero_()
    return c


def test_one_key_over_and_over():
    """Every product of keys is 1: the triangular system at its fullest."""
    check(one_key(1.0))


def test_one_key_turned_over_and_over():
    """With beta 2 a step turns the state's part along the key round and adds 2 v
    to it: nothing fades, and what a chunk adds cancels. Its corrections are w_i
    = sum_j T_ij r_j over up to 64 tokens with |T_ij| <= 2 and |r_j| <= 2 (|v| +
    |column|), and the state gets the sum of 64 of them; with 2^-22 of each term
    (the parts' bits) a chunk's error is at most 64 * 64 * 2 * 2^-22 * 2 (|v| +
    |column|), and the 150 tokens have 3 chunks. Outputs have as much, times
    scale |q| = 1/8."""
    c = one_key(2.0)
    o, states = run(c)
    want_o, want_s, _ = expect(c)
    size = float(c["v"].abs().max()) + np.sqrt((want_s**2).sum(-2)).max() + np.sqrt((c["states"].cpu().numpy() ** 2).sum(-2)).max()
    bound = 3 * 64 * 64 * 2 * 2.0**-22 * 2 * size
    assert np.abs(states.double().cpu().numpy() - want_s).max() <= bound
    assert (np.abs(o.double().cpu().numpy() - want_o) <= torch.finfo(F16).eps / 2 * np.abs(want_o) + bound / 8).all()


@pytest.mark.parametrize("n", [3, 100])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["q", "k", "v", "beta", "log_decay"])
def test_what_is_not_finite_stays_where_it_is(n, bad, where):
    c = case([n, n, n], seed=15, held=[1, 1, 1])
    clean_o, clean_s = run(c)
    at = n + n // 2
    if where in ("beta", "log_decay"):
        c[where][at, 0] = bad
    else:
        c[where][at, 0, 3] = bad
    o, states = run(c)
    assert torch.equal(o[:n], clean_o[:n]) and torch.equal(o[2 * n :], clean_o[2 * n :])
    assert torch.equal(states[0], clean_s[0]) and torch.equal(states[2], clean_s[2])
    assert torch.equal(states[1, 1], clean_s[1, 1]) and torch.equal(o[:, 1], clean_o[:, 1])
    if where == "v":  # the column alone
        keep = [j for j in range(64) if j != 3]
        assert torch.equal(o[..., keep], clean_o[..., keep]) and torch.equal(states[..., keep], clean_s[..., keep])
        assert not torch.isfinite(states[1, 0, :, 3]).any()
    if where == "q":
        assert torch.equal(states, clean_s)
        assert not torch.isfinite(o[at, 0]).any()
    if where == "k":
        assert not torch.isfinite(states[1, 0]).any()


@pytest.mark.parametrize("n", [4, 100])
def test_idle_places_keep_their_states(n):
    c = case([0, n, 0], seed=16, held=[0, 0, 9])
    o, states = check(c)
    assert torch.equal(states[0], c["states"][0]) and torch.equal(states[2], c["states"][2])


def test_rows_of_nobody_are_zero():
    c = case([20, 2], seed=17, lead=6, tail=90)
    o, _ = run(c)
    assert not o[:6].any() and not o[28:].any() and o[6:28].any()
    c = case([2, 2], seed=17, lead=6, tail=90)
    o, _ = run(c, max_query_len=2)
    assert not o[:6].any() and not o[10:].any() and o[6:10].any()


@pytest.mark.parametrize("most", [4, 100])
@pytest.mark.parametrize("offsets", [[0, 30, 20, 40], [-1, 5, 10, 40], [0, 10, 20, 41], [40, 30, 20, 0]])
def test_offsets_out_of_order(most, offsets):
    c = case([10, 10, 20], seed=18)
    c["offsets"] = offsets
    o, states = run(c, most)
    assert not o.any() and torch.equal(states, c["states"])


def test_no_requests_and_no_tokens():
    c = case([], seed=19, tail=9)
    o, _ = run(c, 1)
    assert o.shape == (9, 2, 64) and not o.any()
    o, _ = run(c, 100)
    assert not o.any()
    c = case([0, 0], seed=19)
    o, states = run(c)
    assert o.shape == (0, 2, 64) and torch.equal(states, c["states"])


@pytest.mark.parametrize("n", [3, 80])
def test_slices_and_odd_strides(n):
    """q, k and v as slices of one projection, and as views nothing loads wide."""
    c = case([n], 2, 2, 64, 64, seed=20)
    want = run(c)
    rows = torch.cat([c["q"].flatten(1), c["k"].flatten(1), c["v"].flatten(1)], 1)
    q, k, v = rows.split([128, 128, 256], 1)
    c.update(q=q.unflatten(1, (2, 64)), k=k.unflatten(1, (2, 64)), v=v.unflatten(1, (4, 64)))
    got = run(c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.zeros(n, 2 * 64 + 3, dtype=F16, device="cuda")[:, 3:]
    odd.copy_(c["q"].flatten(1))
    c["q"] = odd.unflatten(1, (2, 64))
    c["k"] = c["k"].transpose(0, 1).contiguous().transpose(0, 1)
    c["v"] = c["v"].transpose(1, 2).contiguous().transpose(1, 2)
    got = run(c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("n", [1, 100])
def test_same_call_same_bits(n):
    c = case([n] * 4, 4, 2, 128, 128, BF16, seed=21)
    first = run(c)
    for _ in range(3):
        again = run(c)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("n", [2, 100])
def test_streams_and_graphs(n):
    """Two calls on streams of their own, and a captured step replayed on new inputs."""
    cases = [case([n, n + 1], 2, 2, 128, 64, seed=22 + i, held=[1, 0]) for i in range(2)]
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            got.append(run(c))
    torch.cuda.synchronize()
    for (o, s), (wo, ws) in zip(got, want):
        assert torch.equal(o, wo) and torch.equal(s, ws)

    fixed = {x: cases[0][x].clone() for x in ("q", "k", "v", "log_decay", "beta", "states")}
    held, offsets = ints(*cases[0]["held"]), ints(*cases[0]["offsets"])
    call = lambda: delta_rule(**fixed, held=held, query_offsets=offsets, max_query_len=n + 1)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = call()
    for c, (wo, ws) in list(zip(cases, want)) * 2:
        for x in fixed:
            fixed[x].copy_(c[x])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, wo) and torch.equal(fixed["states"], ws)
        run(cases[1])


def test_refusals():
    c = case([1, 1], seed=30)
    def call(offsets=None, held=None, most=None, **kw):
        args = {x: c[x] for x in ("q", "k", "v", "log_decay", "beta", "states")}
        args.update(kw)
        return delta_rule(**args, held=held, query_offsets=offsets, max_query_len=most)
    for kw, text in [
        (dict(q=c["q"].float()), "one type"), (dict(q=c["q"].float(), k=c["k"].float(), v=c["v"].float()), "fp16 or bf16"),
        (dict(states=c["states"].double()), "fp32"), (dict(states=c["states"].transpose(2, 3)), "contiguous"),
        (dict(log_decay=c["log_decay"].half()), "log_decay"), (dict(beta=c["beta"][:1]), "beta"),
        (dict(v=c["v"][:, :1]), "v must be"), (dict(k=c["k"][..., :32]), "q and k"),
        (dict(offsets=ints(0, 2)), "query_offsets"), (dict(held=ints(0, 1, 2)), "held"),
        (dict(offsets=ints(0, 1, 2).long()), "query_offsets"), (dict(most=0), "max_query_len"),
        (dict(states=c["states"][:1]), "one token"), (dict(q=c["q"].cpu()), "device"),
        (dict(held=torch.zeros(2, dtype=torch.int32)), "device"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call(**kw)
    small = case([1], 1, 1, 32, 64, seed=31)
    with pytest.raises(RuntimeError, match="64 or 128"):
        run(small)
    three = torch.zeros(2, 3, 64, 64, device="cuda")
    with pytest.raises(RuntimeError, match="multiple"):
        delta_rule(c["q"], c["k"], torch.zeros(2, 3, 64, device="cuda").half(), torch.zeros(2, 3, device="cuda"),
                   torch.zeros(2, 3, device="cuda"), three)


def rows_apart(n, dtype, first, then, log_decay, seed):
    """Requests whose values are `first` in size for 20 tokens of every 50 and
    `then` in the others, with a decay before each change to `then`."""
    c = case([n], 2, 1, 64, 64, dtype, seed=seed, held=[1])
    t = torch.arange(n, device="cuda") % 50
    size = torch.where(t < 20, first, then).view(n, 1, 1)
    c["v"] = (c["v"].float() * size).to(dtype)
    c["log_decay"][t == 20] = log_decay
    return c


@pytest.mark.parametrize("n", [9, 60, 130])
@pytest.mark.parametrize("dtype,first,then,log_decay", [
    (F16, 1e4, 1e-3, -16.0), (F16, 1e4, 1e-3, -float("inf")), (F16, 1e-3, 1e4, 0.0), (BF16, 1e6, 1.0, -14.0), (BF16, 1e12, 1.0, -28.0),
    (BF16, 1e12, 1.0, -float("inf")), (BF16, 1.0, 1e12, 0.0), (BF16, 1e25, 1e-5, -69.0), (BF16, 1e-20, 1e10, -1.0)])
def test_rows_of_values_far_apart(n, dtype, first, then, log_decay):
    """What a decay leaves of large values next to small ones, and small values
    before large ones: a token's error is that of the state as it is then, so
    that the bounds of outputs and states stand as they are."""
    check(rows_apart(n, dtype, first, then, log_decay, seed=35))


@pytest.mark.parametrize("n", [12, 64, 200])
def test_rows_and_decays_of_every_size(n):
    """Values of eight powers of ten, each token's its own, and decays from none to all."""
    c = case([n], 2, 2, 128, 64, BF16, seed=36, held=[1])
    g = torch.Generator().manual_seed(37)
    c["v"] = (c["v"].float() * (10.0 ** (8 * torch.rand(n, 4, 1, generator=g) - 4)).cuda()).to(BF16)
    strong = (torch.rand(n, 4, generator=g) < 0.2).cuda()
    c["log_decay"] = torch.where(strong, -(40 * torch.rand(n, 4, generator=g)).cuda(), c["log_decay"])
    c["log_decay"][(torch.rand(n, 4, generator=g) < 0.03).cuda()] = -float("inf")
    check(c)


@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_one_key_at_beta_two_keeps_what_is_promised(size, dtype):
    """What 64 tokens of one key with beta 2 cost in a chunk: T = (1 + A)^-1 has
    entries of up to 2 throughout, A's are off by four roundings (the key's
    length twice, beta, the product), and a correction goes through up to 64
    rows and 64 columns of them: 64 * 64 * 2 * 4 * 2^-24 = 2e-3 of the values and
    the column, which is what the interface says. Tokens one by one keep 1e-4."""
    for n, most, promised in ((150, None, 2e-3), (150, 1, 1e-4)):
        c = case([n], 2, 1, size, 64, dtype, seed=38, held=[1])
        c["k"][:] = c["k"][:1].clone()
        c["beta"].fill_(2.0)
        c["log_decay"].zero_()
        o, states = run(c, most)
        want_o, want_s, reach = expect(c)
        column = np.sqrt((want_s**2).sum(-2, keepdims=True))
        most_v = np.abs(c["v"].double().cpu().numpy()).max(0)[None, :, None]
        bound = promised * (column + most_v)
        assert (np.abs(states.double().cpu().numpy() - want_s) <= bound).all()
        bound_o = torch.finfo(dtype).eps / 2 * np.abs(want_o) + promised * (reach + most_v[:, :, 0] * size**-0.5) + 2.0**-25
        assert (np.abs(o.double().cpu().numpy() - want_o) <= bound_o).all()


@pytest.mark.parametrize("places", [(0, 1, 2, 3, 4, 5), (63, 64, 127, 128, 400, 699), (694, 695, 696, 697, 698, 699)])
def test_prompts_among_hundreds_of_single_tokens(places):
    """Chunks are numbered by the requests that have any: those before, between and
    behind them take no number."""
    lens = [1] * 700
    for b, n in zip(places, (17, 64, 65, 130, 300, 128)):
        lens[b] = n
    lens[350] = 0
    check(case(lens, 1, 1, 64, 64, BF16, seed=39, lead=60, tail=9), max_query_len=300)


def test_as_many_prompts_as_there_is_room_for():
    """Requests of 17 tokens alone, the most that tokens can be of, and empty ones:
    the numbers' end."""
    check(case([17, 0] * 70, 1, 1, 64, 64, seed=40), max_query_len=17)
    check(case([0, 17, 0], 1, 1, 64, 64, seed=41), max_query_len=17)


def test_a_loose_max_query_len_costs_little():
    """60 prompts of 100 tokens: how long a call takes hardly depends on whether
    max_query_len is the longest, all tokens (its default) or a model's limit. The
    least of several measurements, and a factor of 2 for the machine's own noise;
    where prompts waited for one another it was 3.2 and 6."""
    c = case([100] * 60, 4, 1, 128, 128, BF16, seed=42)
    states, offsets, held = c["states"].clone(), ints(*c["offsets"]), ints(*c["held"])
    args = [c[x] for x in ("q", "k", "v", "log_decay", "beta")]

    def least(most):
        times = []
        for _ in range(6):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(20):
                delta_rule(*args, states, held, offsets, most)
            end.record()
            end.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    least(100)
    exact = least(100)
    assert least(None) < 2 * exact and least(32768) < 2 * exact


@pytest.mark.parametrize("most", [None, 500, 10**6])
def test_workgroups_that_take_several_prompts(most):
    """More prompts than there is room for, of lengths around chunks and with short
    requests between: 50 of 16 heads, where 12 fill the chip three times."""
    lens = [(17, 64, 130, 1, 40, 65, 0, 128)[b % 8] for b in range(64)] + [500]
    check(case(lens, 8, 2, 128, 64, F16, seed=43, lead=2, tail=5), max_query_len=most)
