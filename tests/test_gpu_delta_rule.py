"""The gated delta rule of a batch of sequences, a token each and whole prompts, against the recurrence in 64 bits.

Tolerance: with keys of length one and 0 <= beta <= 1 a token's map of a state row m is no expansion, so the errors of the tokens add up, each at most some 2^-22 (|m| + |v|)
(sums of 16 rounded steps, products of numbers held to 2^-22); they are of either sign, hence a root of their number, four deviations of which are
8 sqrt(T + 16) 2^-22 (max |m| + max |v|), plus half a step of the output's type."""
import math

import numpy as np
import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _inputs(g, T, groups, rank, S, dt, n_slots, gate="mixed", keys="random"):
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(dt)  # noqa: E731
    x = dict(q=unit(rnd(T, groups, S)), k=unit(rnd(T, groups, S)), v=rnd(T, rank, S).to(dt), beta=torch.sigmoid(rnd(T, rank)), state=rnd(n_slots, rank, S, S) * 0.1)
    if keys == "same":                                    # every key the same: what a token corrects is what the one before it wrote
        x["k"] = x["k"][:1].expand(T, groups, S).contiguous()
        x["beta"] = torch.ones_like(x["beta"])
    if keys == "near":
        x["k"] = unit(x["k"][:1].float() + 0.05 * rnd(T, groups, S))
    x["gate"] = {"mixed": -torch.exp(rnd(T, rank) * 1.5 - 2.0), "none": torch.zeros(T, rank, device="cuda"), "strong": -torch.rand(T, rank, generator=g, device="cuda") * 60,
                 "cut": torch.where(torch.rand(T, rank, generator=g, device="cuda") < 0.1, -math.inf, -0.01)}[gate]
    return x


def _reference(x, cu, slots, scale):
    """Rows of out and the states, in 64 bits; a token's map is applied to all heads at once."""
    out, state = torch.zeros(x["v"].shape, dtype=torch.float64, device="cuda"), x["state"].double()
    width = x["v"].shape[1] // x["q"].shape[1]
    most = 0.0
    for b, s in enumerate(slots):
        if s < 0:
            continue
        m = state[s]
        for t in range(cu[b], cu[b + 1]):
            k, q = (x[n][t].double().repeat_interleave(width, 0) for n in ("k", "q"))
            m = m * torch.exp(x["gate"][t].double())[:, None, None]
            d = (x["v"][t].double() - torch.einsum("hij,hj->hi", m, k)) * x["beta"][t].double()[:, None]
            m = m + d[:, :, None] * k[:, None]
            out[t] = torch.einsum("hij,hj->hi", m, q) * scale
        most = max(most, float(m.norm(dim=-1).max()))
        state[s] = m
    return out, state, max(most, float(x["state"].double().norm(dim=-1).max()))


def _close(x, cu, slots, got, state, scale):
    out, want, most = _reference(x, cu, slots, scale)
    T = max(b - a for a, b in zip(cu, cu[1:])) if len(cu) > 1 else 1
    unit = 8 * math.sqrt(T + 16) * 2.0 ** -22 * (most + float(x["v"].double().abs().max()))
    rows = torch.zeros(got.shape[0], dtype=torch.bool, device="cuda")
    for b, s in enumerate(slots):
        if s >= 0:
            rows[cu[b]:cu[b + 1]] = True
    tol = unit * abs(scale) + torch.finfo(got.dtype).eps / 2 * out.abs()
    far = ((got.double() - out).abs() / tol)[rows]
    assert far.numel() == 0 or float(far.max()) <= 1, float(far.max())
    assert bool((got[~rows] == 7.0).all())                # rows of no sequence
    far = ((state.double() - want).abs() / unit)
    assert float(far.max()) <= 1, float(far.max())
    used = [s for s in slots if s >= 0]
    rest = [s for s in range(state.shape[0]) if s not in used]
    assert torch.equal(state[rest], x["state"][rest])


def _rule(x, cu, slots, dims, n_slots, stream=None):
    state, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    cu_d, sl = torch.tensor(cu, dtype=torch.int32, device="cuda"), torch.tensor(slots, dtype=torch.int32, device="cuda")
    T = x["v"].shape[0]
    work = torch.full((dims.workspace(T, len(slots)),), 0xff, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    rc.delta_rule_device(dims, T, len(slots), cu_d.data_ptr(), sl.data_ptr(), n_slots, *[x[n].data_ptr() for n in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(),
                         work.data_ptr(), work.numel(), (stream or torch.cuda.current_stream()).cuda_stream)
    torch.cuda.synchronize()
    return out, state


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups, rank, S", [(16, 32, 128), (2, 6, 64), (1, 1, 32), (3, 3, 128), (2, 8, 256)])
def test_prompts(dtype, groups, rank, S):
    lens = [1, 0, 63, 64, 65, 2, 130, 17, 200]
    cu = np.cumsum([0] + lens).tolist()
    g = _gen(groups * S)
    x = _inputs(g, cu[-1] + 5, groups, rank, S, TYPES[dtype][1], len(lens) + 3)       # five rows behind the last sequence
    slots = [7, 0, 3, 11, 1, -1, 4, 9, 2]
    dims = rc.DeltaDims(TYPES[dtype][0], groups, rank, S)
    out, state = _rule(x, cu, slots, dims, len(lens) + 3)
    _close(x, cu, slots, out, state, 1 / math.sqrt(S))
    rc.device_status()


@pytest.mark.parametrize("S", [64, 128])
@pytest.mark.parametrize("gate", ["none", "strong", "cut"])
@pytest.mark.parametrize("keys", ["random", "same", "near"])
def test_gates_and_keys(S, gate, keys):
    cu = [0, 700]
    x = _inputs(_gen(S), 700, 2, 4, S, torch.float32, 1, gate, keys)
    dims = rc.DeltaDims(0, 2, 4, S)
    _close(x, cu, [0], *_rule(x, cu, [0], dims, 1), 1 / math.sqrt(S))


@pytest.mark.parametrize("T", [3000, 5001])
def test_long_prompts(T):
    cu = [0, T - 1000, T]
    x = _inputs(_gen(T), T, 1, 2, 128, torch.float32, 2)
    _close(x, cu, [1, 0], *_rule(x, cu, [1, 0], rc.DeltaDims(0, 1, 2, 128), 2), 1 / math.sqrt(128))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_scale(dtype):
    """q, k and v as parts of one row, as a projection leaves them."""
    T, groups, rank, S = 150, 2, 4, 128
    dt = TYPES[dtype][1]
    x = _inputs(_gen(1), T, groups, rank, S, dt, 1)
    row = torch.cat([x["q"].flatten(1), x["k"].flatten(1), x["v"].flatten(1)], 1)
    n = row.shape[1]
    y = dict(x, q=row, k=row[:, groups * S:], v=row[:, 2 * groups * S:])
    dims = rc.DeltaDims(TYPES[dtype][0], groups, rank, S, n, n, n, 0.25)
    state, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    work = torch.empty(dims.workspace(T, 1), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    rc.delta_rule_device(dims, T, 1, cu.data_ptr(), 0, 1, *[y[k].data_ptr() for k in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel(),
                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _close(x, [0, T], [0], out, state, 0.25)


def test_large_and_small_states():
    """States, values and keys far from 1: what is held in fewer bits has to be scaled by what is there."""
    for size in (1e-6, 1e5):
        x = _inputs(_gen(2), 300, 1, 2, 128, torch.float32, 1)
        x["v"], x["state"] = x["v"] * size, x["state"] * size
        _close(x, [0, 300], [0], *_rule(x, [0, 300], [0], rc.DeltaDims(0, 1, 2, 128), 1), 1 / math.sqrt(128))
    x = _inputs(_gen(3), 300, 1, 2, 128, torch.float32, 1)
    x["k"], x["beta"], x["q"] = x["k"] * 50.0, x["beta"] / 2500.0, x["q"] * 1e-4
    x["state"] = x["state"] / 50.0
    y = dict(x, k=x["k"] / 50.0, beta=x["beta"] * 2500.0, state=x["state"] * 50.0, q=x["q"] * 1e4)       # the same with keys of length one: S k is the same
    out, state = _rule(x, [0, 300], [0], rc.DeltaDims(0, 1, 2, 128), 1)
    _close(y, [0, 300], [0], out * 50.0 * 1e4, state * 50.0, 1 / math.sqrt(128))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("groups, rank, S", [(16, 32, 128), (2, 6, 64), (1, 3, 32), (2, 4, 256)])
@pytest.mark.parametrize("B", [1, 2, 33])
def test_steps(dtype, groups, rank, S, B):
    x = _inputs(_gen(B), B, groups, rank, S, TYPES[dtype][1], B + 2, "cut")
    slots = torch.randperm(B + 2)[:B].tolist()
    if B > 2:
        slots[3] = -1                                     # a padded row of the batch
    state, out, sl = x["state"].clone(), torch.full_like(x["v"], 7.0), torch.tensor(slots, dtype=torch.int32, device="cuda")
    dims = rc.DeltaDims(TYPES[dtype][0], groups, rank, S)
    torch.cuda.synchronize()
    rc.delta_step_device(dims, B, sl.data_ptr(), B + 2, *[x[n].data_ptr() for n in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _close(x, list(range(B + 1)), slots, out, state, 1 / math.sqrt(S))
    rc.device_status()


@pytest.mark.parametrize("form", ["rule", "step"])
def test_slots_that_cannot_be(form):
    """A slot beyond the states, one below -1, one that an earlier sequence has: reported, the sequences left out, the others served."""
    x = _inputs(_gen(4), 5, 1, 2, 64, torch.float32, 3)
    slots, cu = [1, 3, 1, -2, 0], list(range(6))
    dims = rc.DeltaDims(0, 1, 2, 64)
    if form == "rule":
        out, state = _rule(x, cu, slots, dims, 3)
    else:
        state, out, sl = x["state"].clone(), torch.full_like(x["v"], 7.0), torch.tensor(slots, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        rc.delta_step_device(dims, 5, sl.data_ptr(), 3, *[x[n].data_ptr() for n in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
    with pytest.raises(rc.RedcudaError, match="slot"):
        rc.device_status()
    _close(x, cu, [1, -1, -1, -1, 0], out, state, 1 / 8)


@pytest.mark.parametrize("cu, fine", [([0, 300, 200, 350], [True, False, True]), ([0, 100, 999, 350], [True, False, False]), ([-5, 100, 200, 350], [False, True, True]),
                                      ([0, 100, 100, 400], [True, True, False])])
def test_bounds_that_cannot_be(cu, fine):
    """Bounds that fall, leave the rows or begin below them: reported, those sequences left out."""
    x = _inputs(_gen(5), 350, 1, 2, 128, torch.float32, 3)
    dims = rc.DeltaDims(0, 1, 2, 128)
    out, state = _rule(x, cu, [0, 1, 2], dims, 3)
    with pytest.raises(rc.RedcudaError, match="bounds"):
        rc.device_status()
    for b in range(3):
        if not fine[b]:
            assert torch.equal(state[b], x["state"][b])
        else:
            y = {n: (a[cu[b]:cu[b + 1]] if n != "state" else a[b:b + 1]) for n, a in x.items()}
            if b and cu[b] < max(cu[:b + 1]):             # rows that two sequences claim may hold either's output
                _, want, most = _reference(y, [0, cu[b + 1] - cu[b]], [0], 1.0)
                assert float((state[b] - want[0]).abs().max()) < 1e-4 * most
            else:
                want, st, _ = _reference(y, [0, cu[b + 1] - cu[b]], [0], 1 / math.sqrt(128))
                assert float((state[b] - st[0]).abs().max()) < 1e-4


def test_a_nan_stays_in_its_sequence():
    x = _inputs(_gen(6), 400, 1, 2, 128, torch.float32, 3)
    cu = [0, 130, 260, 400]
    clean, _ = _rule(x, cu, [0, 1, 2], rc.DeltaDims(0, 1, 2, 128), 3)
    x["v"][200, 1, 5] = math.nan
    out, state = _rule(x, cu, [0, 1, 2], rc.DeltaDims(0, 1, 2, 128), 3)
    assert torch.equal(out[:130], clean[:130]) and torch.equal(out[260:], clean[260:])
    assert torch.equal(out[130:200], clean[130:200]) and bool(out[200:260, 1, 5].isnan().all()) and bool(state[1, 1, 5].isnan().all())
    assert bool(state[0].isfinite().all()) and bool(state[2].isfinite().all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what, value", [("q", math.nan), ("k", math.inf), ("k", math.nan), ("gate", math.nan), ("gate", math.inf), ("beta", -math.inf), ("v", math.inf)])
@pytest.mark.parametrize("t", [130, 193, 200, 257])
def test_what_is_not_finite_comes_from_its_token_on(dtype, what, value, t):
    """The tokens before it, also those of its chunk, and the other sequences are as they were to the bit; a query spoils its own output alone."""
    x = _inputs(_gen(6), 400, 1, 2, 128, TYPES[dtype][1], 3)
    cu, dims = [0, 130, 260, 400], rc.DeltaDims(TYPES[dtype][0], 1, 2, 128)
    clean, want = _rule(x, cu, [0, 1, 2], dims, 3)
    x[what][(t, 0, 7) if what in ("q", "k") else (t, 1, 5) if what == "v" else (t, 1)] = value
    out, state = _rule(x, cu, [0, 1, 2], dims, 3)
    heads = {"q": [0, 1], "k": [0, 1]}.get(what, [1])
    last = t + 1 if what == "q" else 260
    for h in (0, 1):
        rows = slice(5, 6) if what == "v" else slice(None)
        if h in heads:
            assert bool(out[t:last, h, rows].isnan().all())
            assert torch.equal(out[:t, h], clean[:t, h]) and torch.equal(out[last:, h], clean[last:, h])
        else:
            assert torch.equal(out[:, h], clean[:, h])
        for s in range(3):
            if s == 1 and h in heads and what != "q":
                assert bool(state[s, h, rows].isnan().all())
                if what == "v":
                    assert torch.equal(state[s, h, :5], want[s, h, :5])
            else:
                assert torch.equal(state[s, h], want[s, h])


def test_capture_and_repeats():
    x = _inputs(_gen(7), 500, 2, 4, 128, torch.bfloat16, 4)
    dims, s = rc.DeltaDims(30, 2, 4, 128), torch.cuda.Stream()
    state, out = x["state"].clone(), torch.zeros_like(x["v"])
    cu, slots = torch.tensor([0, 0, 0, 0], dtype=torch.int32, device="cuda"), torch.tensor([2, 0, 3], dtype=torch.int32, device="cuda")
    work = torch.empty(dims.workspace(500, 3), dtype=torch.uint8, device="cuda")
    call = lambda: rc.delta_rule_device(dims, 500, 3, cu.data_ptr(), slots.data_ptr(), 4, *[x[n].data_ptr() for n in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(),  # noqa: E731
                                        work.data_ptr(), work.numel(), s.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
        for bounds in ([0, 500, 500, 500], [0, 100, 290, 500], [0, 1, 2, 3]):
            cu.copy_(torch.tensor(bounds, dtype=torch.int32))
            state.copy_(x["state"])
            out.fill_(7.0)
            graph.replay()
            s.synchronize()
            got = out.clone(), state.clone()
            _close(x, bounds, [2, 0, 3], *got, 1 / math.sqrt(128))
            state.copy_(x["state"])
            call()
            s.synchronize()
            assert torch.equal(out, got[0]) and torch.equal(state, got[1])
    del graph


def test_prompt_is_its_tokens():
    """A prompt at once, in two pieces, and a token at a time leave the same states and outputs, within the rounding."""
    x = _inputs(_gen(8), 333, 2, 4, 128, torch.float32, 1)
    dims = rc.DeltaDims(0, 2, 4, 128)
    whole, state = _rule(x, [0, 333], [0], dims, 1)
    parts, st = [], x["state"]
    for a, b in ((0, 190), (190, 191), (191, 333)):
        y = {n: t[a:b].contiguous() for n, t in x.items() if n != "state"}
        o, st = _rule(dict(y, state=st), [0, b - a], [0], dims, 1)
        parts.append(o)
    assert float((torch.cat(parts) - whole).abs().max()) <= 2e-5 and float((st - state).abs().max()) <= 2e-5


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_host_form(dtype):
    x = _inputs(_gen(9), 90, 2, 4, 64, torch.float16 if dtype == np.float16 else torch.float32, 3)
    h = {n: t.cpu().numpy() for n, t in x.items()}
    state = h["state"].copy()
    out = rc.delta_rule(h["q"], h["k"], h["v"], h["gate"], h["beta"], state, [0, 30, 90], [2, 0])
    assert out.dtype == dtype
    _close(x, [0, 30, 90], [2, 0], torch.from_numpy(out).cuda(), torch.from_numpy(state).cuda(), 1 / 8)
    with pytest.raises(rc.RedcudaError, match="slot"):
        rc.delta_rule(h["q"], h["k"], h["v"], h["gate"], h["beta"], state, [0, 30, 90], [2, 2])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_keys_and_queries_of_many_sizes(dtype):
    """Tokens whose keys and queries are up to 2^12 apart, some of them zero: an output is as good as its own query is large."""
    x = _inputs(_gen(10), 300, 2, 4, 128, TYPES[dtype][1], 1)
    size = torch.exp2(-torch.randint(0, 13, (2, 300), generator=_gen(11), device="cuda").float())
    size[:, [0, 70, 71, 299]] = 0.0
    x["q"], x["k"] = [(x[n].float() * size[i][:, None, None]).to(x[n].dtype) for i, n in enumerate("qk")]        # powers of two: exact but for what F16 rounds below 2^-14
    out, state = _rule(x, [0, 300], [0], rc.DeltaDims(TYPES[dtype][0], 2, 4, 128), 1)
    assert bool((out[size[0] == 0] == 0).all())
    rows = size[0] > 0
    want, last, most = _reference(x, [0, 300], [0], 1 / math.sqrt(128))
    unit = 8 * math.sqrt(316) * 2.0 ** -22 * (most + float(x["v"].double().abs().max()))
    length = x["q"].double().norm(dim=-1).amax(-1)
    tol = unit / math.sqrt(128) * length[:, None, None] + torch.finfo(out.dtype).eps / 2 * want.abs() + 2.0 ** -25 * (out.dtype == torch.float16)      # half a step of F16's smallest numbers
    assert bool(((out.double() - want).abs() <= tol)[rows].all()), float(((out.double() - want).abs() / tol)[rows].max())
    assert float((state.double() - last).abs().max()) <= unit


@pytest.mark.parametrize("B", [65535, 65536, 70001])
def test_very_many_sequences(B):
    """More sequences than a grid has rows of blocks, a token each: the step and the rule, with some of them padded."""
    x = _inputs(_gen(B), B, 1, 1, 32, torch.float32, B)
    slots = torch.arange(B - 1, -1, -1, dtype=torch.int32, device="cuda")
    slots[5], slots[B - 2] = -1, -1
    state, out, dims = x["state"].clone(), torch.full_like(x["v"], 7.0), rc.DeltaDims(0, 1, 1, 32)
    again, other = x["state"].clone(), torch.full_like(x["v"], 7.0)
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    rows = [x[n].data_ptr() for n in ("q", "k", "v", "gate", "beta")]
    torch.cuda.synchronize()
    s = torch.cuda.current_stream().cuda_stream
    rc.delta_step_device(dims, B, slots.data_ptr(), B, *rows, state.data_ptr(), out.data_ptr(), s)
    rc.delta_rule_device(dims, B, B, cu.data_ptr(), slots.data_ptr(), B, *rows, again.data_ptr(), other.data_ptr(), 0, 0, s)
    torch.cuda.synchronize()
    rc.device_status()
    live = slots >= 0
    k, q, v = (x[n][:, 0].double() for n in ("k", "q", "v"))
    m = x["state"][slots.clamp(min=0).long(), 0].double() * torch.exp(x["gate"].double())[:, :, None]
    m = m + ((v - (m @ k[:, :, None])[:, :, 0]) * x["beta"].double())[:, :, None] * k[:, None]
    unit = 8 * math.sqrt(17) * 2.0 ** -22 * (float(m.norm(dim=-1).max()) + float(v.abs().max()))
    want = (m @ q[:, :, None])[:, :, 0] / math.sqrt(32)
    for st, o in ((state, out), (again, other)):
        assert float((o[:, 0].double() - want)[live].abs().max()) <= unit and bool((o[~live] == 7.0).all())
        assert float((st[slots[live].long(), 0].double() - m[live]).abs().max()) <= unit
        unused = torch.ones(B, dtype=torch.bool, device="cuda")
        unused[slots[live].long()] = False
        assert torch.equal(st[unused], x["state"][unused])


@pytest.mark.parametrize("groups, rank", [(1, 4), (4, 4), (20, 40), (8, 48)])       # few states: several blocks each; many: one each
@pytest.mark.parametrize("gate, keys", [("none", "same"), ("strong", "random"), ("cut", "near"), ("mixed", "same")])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_and_keys_of_few_and_many_heads(groups, rank, gate, keys, dtype):
    cu = [0, 333]
    x = _inputs(_gen(rank), 333, groups, rank, 128, TYPES[dtype][1], 1, gate, keys)
    _close(x, cu, [0], *_rule(x, cu, [0], rc.DeltaDims(TYPES[dtype][0], groups, rank, 128), 1), 1 / math.sqrt(128))


@pytest.mark.parametrize("T", [256, 319, 320, 321, 1000])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_one_sequence(T, dtype):
    """Rows ahead of the sequence and behind it are left as they were."""
    x = _inputs(_gen(T), T + 90, 2, 6, 128, TYPES[dtype][1], 3)
    _close(x, [70, 70 + T], [1], *_rule(x, [70, 70 + T], [1], rc.DeltaDims(TYPES[dtype][0], 2, 6, 128), 3), 1 / math.sqrt(128))


@pytest.mark.parametrize("groups, rank", [(1, 2), (20, 40)])
@pytest.mark.parametrize("what, value", [("q", math.nan), ("k", math.inf), ("gate", math.nan), ("beta", -math.inf), ("v", math.inf), ("v", math.nan)])
@pytest.mark.parametrize("t", [0, 63, 200, 257, 399])
def test_what_is_not_finite_in_one_sequence(groups, rank, what, value, t):
    """As above, where the one sequence's states are worked on by several blocks each, or by one."""
    x = _inputs(_gen(6), 400, groups, rank, 128, torch.float32, 1)
    cu, dims = [0, 400], rc.DeltaDims(0, groups, rank, 128)
    clean, want = _rule(x, cu, [0], dims, 1)
    x[what][(t, 0, 7) if what in ("q", "k") else (t, 1, 37) if what == "v" else (t, 1)] = value
    out, state = _rule(x, cu, [0], dims, 1)
    last = t + 1 if what == "q" else 400
    for h in range(rank):
        if h in ([0, 1] if what in ("q", "k") else [1]):
            rows = slice(37, 38) if what == "v" else slice(None)
            assert bool(out[t:last, h, rows].isnan().all())
            assert torch.equal(out[:t - t % 64, h], clean[:t - t % 64, h]) if what == "q" else torch.equal(out[:t, h], clean[:t, h])
            if what == "q":
                # A chunk's queries share an exponent, which the largest of them sets: without that one the others' lower digits may be rounded at another place. Either output is within its
                # tolerance of the exact one, so they differ by twice that at most; what follows the chunk is the same.
                end = min(400, t - t % 64 + 64)
                unit = 8 * math.sqrt(416) * 2.0 ** -22 * (float(want.norm(dim=-1).max()) + float(x["v"].abs().max())) / math.sqrt(128)
                near = [i for i in range(t - t % 64, end) if i != t]
                assert float((out[near, h] - clean[near, h]).abs().max()) <= 2 * unit and torch.equal(out[end:, h], clean[end:, h])
            else:
                assert torch.equal(out[last:, h], clean[last:, h])
            if what != "q":
                assert bool(state[0, h, rows].isnan().all())
            if what == "v":
                others = [i for i in range(128) if i != 37]
                assert torch.equal(state[0, h][others], want[0, h][others]) and torch.equal(out[:, h][:, others], clean[:, h][:, others])
        else:
            assert torch.equal(out[:, h], clean[:, h]) and torch.equal(state[0, h], want[0, h])


@pytest.mark.parametrize("groups, rank", [(1, 2), (20, 40)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_a_state_that_is_not_finite(groups, rank, value):
    """A row of the state with an infinity or a NaN is no number from the first token on; the other rows are as they were."""
    x = _inputs(_gen(16), 400, groups, rank, 128, torch.float32, 1)
    dims, others = rc.DeltaDims(0, groups, rank, 128), [i for i in range(128) if i != 70]
    clean, want = _rule(x, [0, 400], [0], dims, 1)
    x["state"][0, 1, 70, 3] = value
    out, state = _rule(x, [0, 400], [0], dims, 1)
    assert bool(out[:, 1, 70].isnan().all()) and bool(state[0, 1, 70].isnan().all())
    assert torch.equal(out[:, 1][:, others], clean[:, 1][:, others]) and torch.equal(state[0, 1][others], want[0, 1][others])
    assert torch.equal(out[:, 0], clean[:, 0]) and torch.equal(state[0, 0], want[0, 0])


@pytest.mark.parametrize("groups, rank", [(1, 2), (20, 40)])
def test_rows_of_many_sizes(groups, rank):
    """Rows of values, and of the state, up to 2^12 apart: each as good as it is large."""
    x = _inputs(_gen(17), 300, groups, rank, 128, torch.float32, 1)
    size = torch.exp2(-torch.randint(0, 13, (rank, 128), generator=_gen(18), device="cuda").float())
    x["v"], x["state"] = x["v"] * size, x["state"] * size[:, :, None]
    out, state = _rule(x, [0, 300], [0], rc.DeltaDims(0, groups, rank, 128), 1)
    y = dict(x, v=x["v"] / size, state=x["state"] / size[:, :, None])                  # the rows by themselves, which are independent: powers of two are exact
    _close(y, [0, 300], [0], out / size, state / size[:, :, None], 1 / math.sqrt(128))


def test_capture_of_few_long_sequences():
    """As test_capture_and_repeats, with rows enough for the form that has several blocks a state: replayed with other bounds, padded sequences, and sequences shorter than a chunk."""
    x = _inputs(_gen(19), 700, 2, 4, 128, torch.float16, 4)
    dims, s = rc.DeltaDims(1, 2, 4, 128), torch.cuda.Stream()
    state, out = x["state"].clone(), torch.zeros_like(x["v"])
    cu, slots = torch.tensor([0, 0, 0], dtype=torch.int32, device="cuda"), torch.tensor([2, 0], dtype=torch.int32, device="cuda")
    work = torch.full((dims.workspace(700, 2),), 0xff, dtype=torch.uint8, device="cuda")
    call = lambda: rc.delta_rule_device(dims, 700, 2, cu.data_ptr(), slots.data_ptr(), 4, *[x[n].data_ptr() for n in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(),  # noqa: E731
                                        work.data_ptr(), work.numel(), s.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
        for bounds, who in (([0, 700, 700], [2, 0]), ([0, 0, 700], [1, 3]), ([0, 65, 129], [3, 1]), ([5, 6, 690], [0, 2]), ([0, 350, 700], [-1, 2]), ([0, 0, 0], [2, 0])):
            cu.copy_(torch.tensor(bounds, dtype=torch.int32))
            slots.copy_(torch.tensor(who, dtype=torch.int32))
            state.copy_(x["state"])
            out.fill_(7.0)
            graph.replay()
            s.synchronize()
            got = out.clone(), state.clone()
            _close(x, bounds, who, *got, 1 / math.sqrt(128))
            state.copy_(x["state"])
            call()
            s.synchronize()
            assert torch.equal(out, got[0]) and torch.equal(state, got[1])
    del graph
    rc.device_status()


@pytest.mark.parametrize("cu, fine", [([0, 600, 400, 800], [True, False, True]), ([0, 100, 999, 800], [True, False, False]), ([-5, 100, 500, 800], [False, True, True])])
def test_bounds_that_cannot_be_of_few_long_sequences(cu, fine):
    x = _inputs(_gen(20), 800, 1, 2, 128, torch.float32, 3)
    out, state = _rule(x, cu, [0, 1, 2], rc.DeltaDims(0, 1, 2, 128), 3)
    with pytest.raises(rc.RedcudaError, match="bounds"):
        rc.device_status()
    for b in range(3):
        if not fine[b]:
            assert torch.equal(state[b], x["state"][b])
        elif not any(fine[o] and o != b and cu[o] < cu[b + 1] and cu[b] < cu[o + 1] for o in range(3)):         # of rows that two sequences claim nothing is said
            y = {n: (a[cu[b]:cu[b + 1]] if n != "state" else a[b:b + 1]) for n, a in x.items()}
            T = cu[b + 1] - cu[b]
            _, want, most = _reference(y, [0, T], [0], 1 / math.sqrt(128))
            assert float((state[b].double() - want[0]).abs().max()) <= 8 * math.sqrt(T + 16) * 2.0 ** -22 * (most + float(y["v"].abs().max()))


def test_slots_that_cannot_be_of_few_long_sequences():
    x = _inputs(_gen(22), 1100, 1, 2, 128, torch.bfloat16, 3)
    slots, cu = [1, 3, 1, -2], [0, 500, 700, 900, 1100]
    out, state = _rule(x, cu, slots, rc.DeltaDims(30, 1, 2, 128), 3)
    with pytest.raises(rc.RedcudaError, match="slot"):
        rc.device_status()
    _close(x, cu, [1, -1, -1, -1], out, state, 1 / math.sqrt(128))
