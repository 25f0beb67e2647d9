"""Decode attention over a paged cache and the writing of its pages, against the formulas in 64 bits.

Tolerance of an output, per element, with w the softmax weights: a score is a sum of products whose partial sums are rounded at most 16 times on the way (8 in
a lane or an instruction, 5 across lanes, scale and bias), so it is off by 16 A 2^-24, A = max_p scale sum_i |q_i k_pi|; the exponential adds 8 units; numerator and
denominator take at most N / 4 + 16 further roundings in sequence. Tensor cores may cut where a processor rounds, hence 2^-23:
    |error| <= 2^-23 (2 (16 A + 8) + N / 4 + 16) sum_p w_p |v_p| + eps / 2 |out|
lse likewise without the factor 2, plus its own rounding."""
import math

import numpy as np
import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]      # queries, cache


class Cache:
    """A pool whose unused rows are NaN, in one of two orders, with a table of scattered pages."""

    def __init__(self, g, cache, n_kv, hd, page, lens, order="dense", spare=3):
        self.type, self.dtype = TYPES[cache]
        need = [-(-max(n, 0) // page) for n in lens]
        self.n_pages, self.width, self.page, self.n_kv, self.hd = sum(need) + spare, max(1, max(need)), page, n_kv, hd
        shape = (self.n_pages, page, n_kv, hd) if order == "dense" else (self.n_pages, n_kv, page, hd)
        pools = [torch.full(shape, math.nan, device="cuda", dtype=self.dtype) for _ in range(2)]
        self.k, self.v = pools if order == "dense" else [p.transpose(1, 2) for p in pools]         # [page][position][head][value] either way
        strides = (0, 0, 0) if order == "dense" else tuple(self.k.stride()[:3])
        perm = torch.randperm(self.n_pages, generator=g, device="cuda").cpu().tolist()
        table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            for i, p in enumerate(perm[at:at + n]):
                rows = min(page, lens[b] - i * page)
                for pool in (self.k, self.v):
                    pool[p, :rows] = torch.randn(rows, n_kv, hd, generator=g, device="cuda").to(self.dtype)
            at += n
        self.spare = perm[at:]
        self.table = table.cuda()
        self.kv = rc.PagedKv(self.type, n_kv, hd, page, self.n_pages, self.k.data_ptr(), self.v.data_ptr(), *strides)

    def rows(self, b, n):
        """K and V of the first n positions of sequence b, in 64 bits, [n][n_kv][hd]; positions without a page left out."""
        p = torch.arange(n)
        pages = self.table[b].cpu().long()[p // self.page]
        keep = (pages >= 0) & (pages < self.n_pages)
        return [x[pages[keep].cuda(), (p % self.page)[keep].cuda()].double() for x in (self.k, self.v)]


def _attend(c, q, lens, n_q, qt, new=None, scale=0.0, q_stride=0, new_stride=0, stream=None):
    B, dt = len(lens), TYPES[qt][1]
    out = torch.full((B, n_q, c.hd), 7.0, device="cuda", dtype=dt)
    lse = torch.full((B, n_q), 7.0, device="cuda")
    work = torch.full((c.kv.attend_workspace(n_q),), 0xff, device="cuda", dtype=torch.uint8)          # what it holds before does not matter
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s = (stream or torch.cuda.current_stream()).cuda_stream
    torch.cuda.synchronize()
    c.kv.attend_device(c.table.data_ptr(), c.width, B, ln.data_ptr(), n_q, TYPES[qt][0], q.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel(), s, scale,
                       new[0].data_ptr() if new else 0, new[1].data_ptr() if new else 0, lse.data_ptr(), q_stride, new_stride)
    torch.cuda.synchronize()
    return out, lse


def _check(c, q, lens, n_q, out, lse, scale=None):
    scale = scale or 1.0 / math.sqrt(c.hd)
    G, eps = n_q // c.n_kv, torch.finfo(out.dtype).eps
    for b, n in enumerate(lens):
        k, v = c.rows(b, max(n, 0))
        if k.shape[0] == 0:
            assert torch.equal(out[b], torch.zeros_like(out[b])) and bool((lse[b] == -math.inf).all()), b
            continue
        k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        x = torch.einsum("hd,phd->hp", q[b].double(), k) * scale
        A = (torch.einsum("hd,phd->hp", q[b].double().abs(), k.abs()) * abs(scale)).amax(-1)
        w = torch.softmax(x, -1)
        want, unit = torch.einsum("hp,phd->hd", w, v), torch.einsum("hp,phd->hd", w, v.abs())
        N = k.shape[0]
        tol = 2.0 ** -23 * (2 * (16 * A + 8) + N / 4 + 16)[:, None] * unit + eps / 2 * want.abs() + torch.finfo(out.dtype).tiny
        assert bool(((out[b].double() - want).abs() <= tol).all()), (b, n, float(((out[b].double() - want).abs() / tol).max()))
        ref = torch.logsumexp(x, -1)
        tol = 2.0 ** -23 * (16 * A + 8 + N / 4 + 16 + ref.abs())
        assert bool(((lse[b].double() - ref).abs() <= tol).all()), (b, n)


def _q(g, B, n_q, hd, qt, scale=1.5):
    return (torch.randn(B, n_q, hd, generator=g, device="cuda") * scale).to(TYPES[qt][1])


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("qt, cache", PAIRS)
@pytest.mark.parametrize("n_q, n_kv, hd", [(16, 2, 256), (8, 8, 64), (32, 8, 128), (24, 2, 128), (17, 1, 64), (3, 3, 256), (40, 8, 128)])
def test_lengths_and_heads(qt, cache, n_q, n_kv, hd):
    lens = [1, 2, 0, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 100, 129, -3, 300, 517]
    g = _gen(n_q * 100 + hd)
    c = Cache(g, cache, n_kv, hd, 16, lens)
    q = _q(g, len(lens), n_q, hd, qt)
    _check(c, q, lens, n_q, *_attend(c, q, lens, n_q, qt))
    rc.device_status()


@pytest.mark.parametrize("qt, cache", PAIRS)
@pytest.mark.parametrize("page", [1, 5, 64, 100, 1000])
@pytest.mark.parametrize("order", ["dense", "heads first"])
def test_pages_and_orders(qt, cache, page, order):
    lens = [211, 1, 640, 0, 99, 1000]
    g = _gen(page)
    c = Cache(g, cache, 2, 128, page, lens, order)
    q = _q(g, len(lens), 12, 128, qt)
    _check(c, q, lens, 12, *_attend(c, q, lens, 12, qt))


@pytest.mark.parametrize("qt, cache", PAIRS)
@pytest.mark.parametrize("lens", [[5000], [20011, 3], [1] * 700, [0] * 5, [0, 0, 0, 1], [4000] * 37, [0] * 300 + [999] + [0] * 300])
def test_splits(qt, cache, lens):
    """Few long sequences, many short ones, empty ones: runs that end inside a head, at its end, and none at all."""
    g = _gen(len(lens))
    c = Cache(g, cache, 2, 64, 64, lens)
    q = _q(g, len(lens), 16, 64, qt)
    _check(c, q, lens, 16, *_attend(c, q, lens, 16, qt))


@pytest.mark.parametrize("qt, cache", PAIRS)
@pytest.mark.parametrize("n_q, n_kv, hd", [(16, 2, 256), (8, 8, 64), (5, 1, 128), (12, 1, 64)])
def test_few_heads(qt, cache, n_q, n_kv, hd):
    """A sequence or a few of every length up to some hundred, in the form for few heads and, by a wide page table, in the other: the same within the tolerance."""
    g = _gen(n_q)
    for lens in ([1], [7], [16], [0], [23], [130], [257], [600], [3, 0, 190], [64, 65, 63]):
        c = Cache(g, cache, n_kv, hd, 16, lens)
        q = _q(g, len(lens), n_q, hd, qt)
        _check(c, q, lens, n_q, *_attend(c, q, lens, n_q, qt))
        wide = torch.full((len(lens), 4000), -1, dtype=torch.int32, device="cuda")
        wide[:, :c.width] = c.table
        c.table, c.width = wide, 4000
        _check(c, q, lens, n_q, *_attend(c, q, lens, n_q, qt))
    rc.device_status()


@pytest.mark.parametrize("qt, cache", PAIRS)
@pytest.mark.parametrize("lens", [[1, 16, 17, 0, 700, 33, 64], [1, 16, 17, 0, 300, 33, 64], [33], [4000, 2]])
def test_new_rows(qt, cache, lens):
    """The new rows are written to the last position and attended to; nothing else of the cache changes."""
    g = _gen(3)
    c = Cache(g, cache, 2, 256, 16, lens)
    dt = TYPES[qt][1]
    new = [torch.randn(len(lens), 5, 256, generator=g, device="cuda").to(dt) for _ in range(2)]       # rows of which the first two heads are meant
    before = [x.clone() for x in (c.k, c.v)]
    q = torch.randn(len(lens), 20, 256, generator=g, device="cuda").to(dt)
    out, lse = _attend(c, q, lens, 16, qt, new, q_stride=20 * 256, new_stride=5 * 256)
    _check(c, q[:, :16], lens, 16, out, lse)
    for x, old, rows in zip((c.k, c.v), before, new):
        for b, n in enumerate(lens):
            if n:
                old[int(c.table[b, (n - 1) // 16]), (n - 1) % 16] = rows[b, :2].to(old.dtype)
        assert torch.equal(x.nan_to_num(99.0), old.nan_to_num(99.0))


@pytest.mark.parametrize("qt, cache", PAIRS)
def test_scale_and_large_scores(qt, cache):
    """Scores of some hundreds: all weight on one position, and the maximum moves along the length."""
    lens = [300, 77]
    g = _gen(5)
    c = Cache(g, cache, 1, 64, 16, lens)
    q = _q(g, 2, 8, 64, qt, 1.0)
    for scale in (4.0, -2.0, 1e-3):
        _check(c, q, lens, 8, *_attend(c, q, lens, 8, qt, scale=scale), scale=scale)


@pytest.mark.parametrize("qt, cache", PAIRS)
def test_wide_values(qt, cache):
    """Queries far from 1 (beyond half precision where they are floats) over keys that bring the scores back, and values of every size."""
    lens = [200]
    g = _gen(6)
    c = Cache(g, cache, 1, 128, 32, lens)
    big = 1e6 if qt == "f32" else 500.0
    q = _q(g, 1, 8, 128, qt, big)
    q[0, 1] *= 1e-9 if qt == "f32" else 1e-3
    q[0, 2] = 0
    _check(c, q, lens, 8, *_attend(c, q, lens, 8, qt, scale=1.0 / big), scale=1.0 / big)


def test_pages_outside_the_cache():
    """Positions whose page is not there are left out and reported, a length beyond the table as well; the cache is not written."""
    lens = [100, 40, 64]
    g = _gen(7)
    c = Cache(g, "f16", 2, 64, 16, lens)
    c.table[0, 2], c.table[1, 1], c.table[2, 3] = -1, c.n_pages, 0x7fffffff
    before = c.k.clone()
    new = [torch.randn(3, 2, 64, device="cuda") for _ in range(2)]
    q = _q(g, 3, 8, 64, "f32")
    out, lse = _attend(c, q, lens, 8, "f32")
    _check(c, q, lens, 8, out, lse)
    with pytest.raises(rc.RedcudaError, match="page"):
        rc.device_status()
    rc.device_status()                                    # cleared
    out, lse = _attend(c, q, [100, 40, 200], 8, "f32", new)
    with pytest.raises(rc.RedcudaError, match="page"):
        rc.device_status()
    before[int(c.table[0, 6]), 3] = new[0][0].half()      # the one new row that has a page and a position in the table
    before[int(c.table[1, 2]), 7] = new[0][1].half()
    assert torch.equal(c.k.nan_to_num(99.0), before.nan_to_num(99.0))


def test_infinity_beyond_the_end_and_inside():
    lens = [20, 20]
    g = _gen(8)
    c = Cache(g, "f32", 1, 64, 16, lens)
    c.v[int(c.table[0, 1]), 4:] = math.inf
    c.k[int(c.table[0, 1]), 4:] = -math.inf
    c.k[int(c.table[1, 0]), 3, 0, 5] = math.nan            # a row that is attended to
    q = _q(g, 2, 8, 64, "f32")
    out, lse = _attend(c, q, lens, 8, "f32")
    assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all())
    c.k[int(c.table[1, 0]), 3, 0, 5] = 0.5
    out, lse = _attend(c, q, lens, 8, "f32")
    _check(c, q, lens, 8, out, lse)


def test_capture_streams_and_repeats():
    """Captured once, replayed with other lengths; the same to the bit as a plain call, on a stream of its own, every time."""
    g = _gen(9)
    c = Cache(g, "bf16", 2, 128, 32, [900, 900, 900])
    q = _q(g, 3, 16, 128, "bf16")
    lens, out, lse = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 16, 128, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 16, device="cuda")
    work = torch.empty(c.kv.attend_workspace(16), device="cuda", dtype=torch.uint8)
    s = torch.cuda.Stream()
    call = lambda: c.kv.attend_device(c.table.data_ptr(), c.width, 3, lens.data_ptr(), 16, 30, q.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel(), s.cuda_stream,  # noqa: E731
                                      lse_ptr=lse.data_ptr())
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call()
        for n in ([900, 1, 0], [5, 700, 311], [0, 0, 0], [64, 32, 33]):
            lens.copy_(torch.tensor(n, dtype=torch.int32))
            out.fill_(3.0)
            graph.replay()
            s.synchronize()
            got = out.clone(), lse.clone()
            _check(c, q, n, 16, *got)
            for _ in range(3):
                call()
                s.synchronize()
                assert torch.equal(out, got[0]) and torch.equal(lse, got[1])
    del graph


def test_far_pages():
    """A pool of more than 2^32 bytes, and of more than 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 30e9:
        pytest.skip("not enough memory")
    n_pages, page = 70000, 64
    k, v = (torch.empty(n_pages, page, 2, 256, dtype=torch.float16, device="cuda") for _ in range(2))
    assert k.numel() > 2 ** 31
    kv = rc.PagedKv(1, 2, 256, page, n_pages, k.data_ptr(), v.data_ptr())
    g = _gen(10)
    table = torch.tensor([[69999, 5, 42000, 69998]], dtype=torch.int32, device="cuda")
    rows = torch.randn(2, 200, 2, 256, generator=g, device="cuda")
    start = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    s = torch.cuda.current_stream().cuda_stream
    kv.append_device(table.data_ptr(), 4, 1, start.data_ptr(), 200, cu.data_ptr(), 0, rows[0].data_ptr(), rows[1].data_ptr(), s)
    c = Cache.__new__(Cache)
    c.k, c.v, c.table, c.page, c.n_pages, c.n_kv, c.hd, c.width, c.kv = k, v, table, page, n_pages, 2, 256, 4, kv
    got = c.rows(0, 200)
    assert torch.equal(got[0], rows[0].half().double()) and torch.equal(got[1], rows[1].half().double())
    q = _q(g, 1, 16, 256, "f32")
    _check(c, q, [200], 16, *_attend(c, q, [200], 16, "f32"))


@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd, order", [(64, "dense"), (256, "heads first")])
def test_append(cache, rows, hd, order):
    """Ragged prompts, an empty one, one that is left out, rows behind the last; values that the cache's type rounds or cannot hold."""
    g = _gen(11)
    lens, start = [5, 0, 40, 1, 17], [3, 9, 0, 16, -1]
    c = Cache(g, cache, 3, hd, 8, [a + n for a, n in zip(start, lens)], order)
    new = [torch.randn(70, 4, hd, generator=g, device="cuda").to(TYPES[rows][1]) for _ in range(2)]       # 7 rows behind the last sequence, 4 heads of which 3 are meant
    new[0][0, 0, :4] = torch.tensor([1e30, -1e30, math.inf, math.nan])
    want = [x.clone() for x in (c.k, c.v)]
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    st = torch.tensor(start, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    c.kv.append_device(c.table.data_ptr(), c.width, 5, st.data_ptr(), 70, cu.data_ptr(), TYPES[rows][0], new[0].data_ptr(), new[1].data_ptr(), torch.cuda.current_stream().cuda_stream, 4 * hd)
    torch.cuda.synchronize()
    t = 0
    for b, n in enumerate(lens):
        for i in range(n):
            if start[b] >= 0:
                p = start[b] + i
                for x, r in zip(want, new):
                    x[int(c.table[b, p // 8]), p % 8] = r[t, :3].to(x.dtype)
            t += 1
    for x, w in zip((c.k, c.v), want):
        assert torch.equal(x.isnan(), w.isnan()) and torch.equal(x.nan_to_num(1.0, 2.0, 3.0), w.nan_to_num(1.0, 2.0, 3.0))
    rc.device_status()


def test_append_one_row_each_and_bad_tables():
    g = _gen(12)
    c = Cache(g, "f16", 2, 64, 4, [9, 9, 9, 9])
    new = [torch.randn(4, 2, 64, generator=g, device="cuda") for _ in range(2)]
    want = c.k.clone()
    c.table[1, 1] = c.n_pages
    st = torch.tensor([8, 5, 12, 0], dtype=torch.int32, device="cuda")        # the second has no page, the third lies beyond the table
    torch.cuda.synchronize()
    s = torch.cuda.current_stream().cuda_stream
    c.kv.append_device(c.table.data_ptr(), c.width, 4, st.data_ptr(), 4, 0, 0, new[0].data_ptr(), new[1].data_ptr(), s)
    torch.cuda.synchronize()
    want[int(c.table[0, 2]), 0], want[int(c.table[3, 0]), 0] = new[0][0].half(), new[0][3].half()
    assert torch.equal(c.k.nan_to_num(9.0), want.nan_to_num(9.0))
    with pytest.raises(rc.RedcudaError, match="page"):
        rc.device_status()
    cu = torch.tensor([0, 3, 1, 4, 4], dtype=torch.int32, device="cuda")      # bounds that do not ascend
    c.kv.append_device(c.table.data_ptr(), c.width, 4, torch.zeros_like(st).data_ptr(), 4, cu.data_ptr(), 0, new[0].data_ptr(), new[1].data_ptr(), s)
    torch.cuda.synchronize()
    try:
        rc.device_status()
    except rc.RedcudaError as e:
        assert "bounds" in str(e) or "page" in str(e)


@pytest.mark.parametrize("n_seqs", [1, 2, 31, 32, 33, 1000, 1025])
def test_append_finds_every_sequence(n_seqs):
    """Bounds of many sequences, most of them of one row, some empty."""
    rng = np.random.default_rng(n_seqs)
    lens = rng.choice([0, 1, 1, 2, 5], n_seqs).tolist()
    lens[-1] += 1
    T = sum(lens)
    k, v = (torch.zeros(n_seqs, 8, 1, 64, device="cuda") for _ in range(2))
    kv = rc.PagedKv(0, 1, 64, 8, n_seqs, k.data_ptr(), v.data_ptr())
    table = torch.arange(n_seqs, dtype=torch.int32, device="cuda")[:, None].contiguous()
    rows = torch.arange(1, T + 1, device="cuda", dtype=torch.float32)[:, None].expand(T, 64).contiguous()
    cu = torch.tensor([0] + lens, device="cuda").cumsum(0).int()
    st = torch.zeros(n_seqs, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    kv.append_device(table.data_ptr(), 1, n_seqs, st.data_ptr(), T, cu.data_ptr(), 0, rows.data_ptr(), rows.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    want = np.zeros((n_seqs, 8), np.float32)
    t = 1
    for b, n in enumerate(lens):
        want[b, :n] = np.arange(t, t + n)
        t += n
    assert np.array_equal(k[:, :, 0, 0].cpu().numpy(), want) and np.array_equal(v[:, :, 0, 63].cpu().numpy(), want)


@pytest.mark.parametrize("qt, cache", PAIRS)
def test_queries_and_rows_of_zeros(qt, cache):
    """Queries of zeros weigh every position alike; keys and values of zeros; queries near the smallest numbers."""
    c = Cache(_gen(14), cache, 2, 128, 16, [200, 33, 5])
    q = _q(_gen(15), 3, 8, 128, qt)
    q[0], q[1, 3] = 0.0, 0.0
    q[2] = (q[2].float() * 2.0 ** -20).to(q.dtype)
    c.k[int(c.table[1, 0])] = 0.0
    c.v[int(c.table[1, 1])] = 0.0
    out, lse = _attend(c, q, [200, 33, 5], 8, qt)
    _check(c, q, [200, 33, 5], 8, out, lse)
