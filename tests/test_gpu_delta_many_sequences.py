"""The gated delta rule in chunks over many sequences, and over bounds of which some cannot be: every sequence whose own bounds ascend within the rows, and whose rows no other has, is
computed; the others are reported and left as they were.

Tolerance as in test_gpu_delta_rule.py: 8 sqrt(T + 16) 2^-22 (max |m| + max |v|) for a state, the same times the scale plus half a step of the type for an output."""
import math

import numpy as np
import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
S = 128


def _inputs(seed, T, groups, rank, dt, n_slots):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(dt)  # noqa: E731
    return dict(q=unit(rnd(T, groups, S)), k=unit(rnd(T, groups, S)), v=rnd(T, rank, S).to(dt), gate=-torch.exp(rnd(T, rank) * 1.5 - 2.0), beta=torch.sigmoid(rnd(T, rank)),
                state=rnd(n_slots, rank, S, S) * 0.1)


def _reference(x, begin, lens, slots):
    """Rows of out and the states of the sequences `slots`, all sequences a token further at a time, in 64 bits."""
    order = sorted(range(len(lens)), key=lambda b: -lens[b])
    begin, lens, slots = ([a[b] for b in order] for a in (begin, lens, slots))
    width = x["v"].shape[1] // x["q"].shape[1]
    m, out, alive = x["state"][slots].double(), torch.zeros(x["v"].shape, dtype=torch.float64, device="cuda"), len(lens)
    first = torch.tensor(begin, device="cuda")
    for t in range(max(lens)):
        while lens[alive - 1] <= t:
            alive -= 1
        at = first[:alive] + t
        k, q = (x[n][at].double().repeat_interleave(width, 1) for n in ("k", "q"))
        y = m[:alive] * torch.exp(x["gate"][at].double())[..., None, None]
        d = (x["v"][at].double() - (y @ k[..., None])[..., 0]) * x["beta"][at].double()[..., None]
        m[:alive] = y + d[..., None] * k[:, :, None]
        out[at] = (m[:alive] @ q[..., None])[..., 0] / math.sqrt(S)
    return out, m, slots


def _workspace(dims, T, n):
    """A workspace whose bytes are all ones: NaN as numbers, and nothing that a call may go by."""
    work = torch.full((dims.workspace(T, n),), 0xff, dtype=torch.uint8, device="cuda")
    assert work.numel()                                   # the form in chunks
    return work


def _call(x, cu, slots, dims, work, state, out):
    cu_d, sl = torch.tensor(cu, dtype=torch.int32, device="cuda"), torch.tensor(slots, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    rc.delta_rule_device(dims, x["v"].shape[0], len(slots), cu_d.data_ptr(), sl.data_ptr(), state.shape[0], *[x[n].data_ptr() for n in ("q", "k", "v", "gate", "beta")], state.data_ptr(),
                         out.data_ptr(), work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()


def _check(x, cu, slots, served, state, out):
    """The sequences `served` against the recurrence; every other row and state as it was."""
    n_slots = x["state"].shape[0]
    lens = [cu[b + 1] - cu[b] for b in served]
    want, m, where = _reference(x, [cu[b] for b in served], lens, [slots[b] for b in served])
    most = max(float(m.norm(dim=-1).max()), float(x["state"].double().norm(dim=-1).max()))
    unit = 8 * math.sqrt(max(lens) + 16) * 2.0 ** -22 * (most + float(x["v"].double().abs().max()))
    rows = torch.zeros(out.shape[0], dtype=torch.bool, device="cuda")
    for b in served:
        rows[cu[b]:cu[b + 1]] = True
    far = ((out.double() - want).abs() / (unit / math.sqrt(S) + torch.finfo(out.dtype).eps / 2 * want.abs()))[rows]
    assert float(far.max()) <= 1, float(far.max())
    assert bool((out[~rows] == 7.0).all())
    far = (state[where].double() - m).abs() / unit
    assert float(far.max()) <= 1, float(far.max())
    rest = torch.ones(n_slots, dtype=torch.bool, device="cuda")
    rest[where] = False
    assert torch.equal(state[rest], x["state"][rest])


ONE_OF_64 = [50 * b if b != 32 else 1000000 for b in range(65)]


@pytest.mark.parametrize("T, cu", [(350, [0, 100, 200, -1, 300]), (350, [0, 100, 200, 50, 9999]), (200, [0, 100, 200, 0, 0]), (300, [200, 300, 0, 100]), (1200, [0, 400, 800, -1, 1100]),
                                   (1200, [0, 400, 800, 9999, 1200]), (1300, [700, 1300, 0, 500]), (3200, ONE_OF_64)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bad_bounds_leave_the_others(dtype, T, cu):
    n = len(cu) - 1
    x, y = (_inputs(s, T, 1, 2, TYPES[dtype][1], n + 1) for s in (1, 2))
    dims = rc.DeltaDims(TYPES[dtype][0], 1, 2, S)
    work = _workspace(dims, T, n)
    _call(y, [min(T, -(-T // n) * b) for b in range(n + 1)], list(range(n)), dims, work, y["state"].clone(), torch.empty_like(y["v"]))
    rc.device_status()
    fine = [b for b in range(n) if 0 <= cu[b] < cu[b + 1] <= T]
    served = [b for b in fine if not any(o != b and cu[o] < cu[b + 1] and cu[b] < cu[o + 1] for o in fine)]
    state, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    _call(x, cu, list(range(n)), dims, work, state, out)
    with pytest.raises(rc.RedcudaError, match="bounds"):
        rc.device_status()
    assert served == fine and len(served) >= 2            # of rows that two claim nothing would be said
    _check(x, cu, list(range(n)), served, state, out)


@pytest.mark.parametrize("T, cu", [(300, [0, 300, 0, 300, 0, 300]), (3000, [0, 3000] * 20)])
def test_rows_that_many_claim(T, cu):
    """More chunks than the call's rows can have: what has no room is left out and reported, and states that no sequence has are not touched."""
    n = len(cu) - 1
    x = _inputs(3, T, 1, 1, torch.float32, n + 2)
    dims = rc.DeltaDims(0, 1, 1, S)
    state, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    _call(x, cu, list(range(n)), dims, _workspace(dims, T, n), state, out)
    with pytest.raises(rc.RedcudaError, match="bounds"):
        rc.device_status()
    bad = [b for b in range(n) if cu[b + 1] < cu[b]] + [n, n + 1]
    assert torch.equal(state[bad], x["state"][bad])


@pytest.mark.parametrize("n", [31, 32, 33, 64, 385, 400, 1024, 1025, 1100])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_sequences(dtype, n):
    rng = np.random.default_rng(n)
    lens = rng.choice([0, 1, 30, 63, 64, 65, 70, 130], n).tolist()
    lens[-1] = 65
    cu = np.cumsum([0] + lens).tolist()
    T = max(cu[-1] + 3, 24 * n + 32)                      # rows behind the last sequence
    slots = rng.permutation(n + 2)[:n].tolist()
    x = _inputs(n, T, 1, 1, TYPES[dtype][1], n + 2)
    dims = rc.DeltaDims(TYPES[dtype][0], 1, 1, S)
    state, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    _call(x, cu, slots, dims, _workspace(dims, T, n), state, out)
    rc.device_status()
    _check(x, cu, slots, [b for b in range(n) if lens[b]], state, out)


def test_more_sequences_than_a_grid_has_rows():
    """65536 sequences and some, 25 tokens each: the states go in two launches. Some of them against the recurrence, among them the last ones of the first launch and all of the second."""
    n, each = 65600, 25
    T = n * each
    x = _inputs(5, T, 1, 1, torch.bfloat16, n)
    dims = rc.DeltaDims(30, 1, 1, S)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda") * each
    state, out = x["state"].clone(), torch.full_like(x["v"], 7.0)
    work = _workspace(dims, T, n)
    torch.cuda.synchronize()
    rc.delta_rule_device(dims, T, n, cu.data_ptr(), 0, n, *[x[a].data_ptr() for a in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel(),
                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    rc.device_status()
    some = [0, 1, 2, 1023, 1024, 40000, 65533, 65534, 65535, 65536] + list(range(65540, n))
    want, m, where = _reference(x, [b * each for b in some], [each] * len(some), some)
    unit = 8 * math.sqrt(each + 16) * 2.0 ** -22 * (max(float(m.norm(dim=-1).max()), float(x["state"][some].double().norm(dim=-1).max())) + float(x["v"].abs().max()))
    assert float((state[where].double() - m).abs().max()) <= unit
    rows = torch.cat([torch.arange(b * each, b * each + each) for b in some]).cuda()
    assert bool(((out[rows].double() - want[rows]).abs() <= unit / math.sqrt(S) + torch.finfo(out.dtype).eps / 2 * want[rows].abs()).all())
    assert not bool((out == 7.0).all(-1).any())           # every row is written


def test_a_sequence_costs_the_same_among_many():
    """The time of a call goes with its sequences: 1000 of them once took six times as long as 1100, as every block of the former looked at all of them for its own place. Twice is allowed here."""
    def time_of(n):
        x = _inputs(6, 64 * n, 4, 8, torch.bfloat16, n)
        dims = rc.DeltaDims(30, 4, 8, S)
        cu, out = torch.arange(n + 1, dtype=torch.int32, device="cuda") * 64, torch.empty_like(x["v"])
        work = _workspace(dims, 64 * n, n)
        torch.cuda.synchronize()
        times = []
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            rc.delta_rule_device(dims, 64 * n, n, cu.data_ptr(), 0, n, *[x[y].data_ptr() for y in ("q", "k", "v", "gate", "beta")], x["state"].data_ptr(), out.data_ptr(), work.data_ptr(),
                                 work.numel(), torch.cuda.current_stream().cuda_stream)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        rc.device_status()
        return sorted(times[1:])[2] / n

    assert time_of(1000) <= 2 * time_of(1100)


@pytest.mark.parametrize("n", [20, 40])
def test_replayed_with_other_bounds(n):
    """A captured call follows its bounds: ragged, most sequences empty, one with every row, some that cannot be, none with a row, and ragged again, all over the same workspace."""
    T = 24 * n + 200
    x = _inputs(7, T, 2, 4, torch.float32, n)
    dims = rc.DeltaDims(0, 2, 4, S)
    slots = list(range(n - 1, -1, -1))
    cu, sl = torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.tensor(slots, dtype=torch.int32, device="cuda")
    state, out, work = x["state"].clone(), torch.full_like(x["v"], 7.0), _workspace(dims, T, n)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        rc.delta_rule_device(dims, T, n, cu.data_ptr(), sl.data_ptr(), n, *[x[y].data_ptr() for y in ("q", "k", "v", "gate", "beta")], state.data_ptr(), out.data_ptr(), work.data_ptr(),
                             work.numel(), stream.cuda_stream)
    ragged = np.sort(np.random.default_rng(n).integers(0, T + 1, n + 1)).tolist()
    bad = [24 * b for b in range(n + 1)]
    bad[3], bad[n - 4] = T + 1, -1
    for bounds in (ragged, [0] * (n - 2) + [70, 70, 199], [0] * 5 + [T] * (n - 4), bad, [T] * (n + 1), ragged):
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        state.copy_(x["state"])
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        served = [b for b in range(n) if 0 <= bounds[b] < bounds[b + 1] <= T]
        if bounds is bad:
            with pytest.raises(rc.RedcudaError, match="bounds"):
                rc.device_status()
        else:
            rc.device_status()
        if served:
            _check(x, bounds, slots, served, state, out)
        else:
            assert torch.equal(state, x["state"]) and bool((out == 7.0).all())
    del graph
