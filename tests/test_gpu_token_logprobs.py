"""Log probabilities, entropies and alternatives of rows of logits against 64 bits.

Tolerance: a thread adds up at most vocab / 256 terms in sequence, each with an exponential of 2 units and an argument d = x - m rounded to |d| 2^-24; joining takes 16 more
steps. The relative error of sum e^d is then at most e = 2^-24 (vocab / 256 + 40 + sum p |d|), that of log its own and as much again; u = sum e^d d likewise with |d| as weight:
    |lp error| <= e + 2^-24 (|lp| + |d|) * 2,    |entropy error| <= e (1 + 2 sum p |d|) + 2^-23 entropy.
Ids are exact: the largest values, the lower id first among equal ones."""
import math

import numpy as np
import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}


def _call(x, tokens, top_n, vocab=None, stride=0, want=("lp", "ent", "top"), stream=None):
    rows, dt = x.shape[0], {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[x.dtype]
    vocab = vocab or x.shape[1]
    lp, ent = torch.full((rows,), 7.0, device="cuda"), torch.full((rows,), 7.0, device="cuda")
    ids, top = torch.full((rows, top_n), 77, dtype=torch.int32, device="cuda"), torch.full((rows, top_n), 7.0, device="cuda")
    tok = None if tokens is None else torch.as_tensor(tokens, dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    rc.token_logprobs_device(dt, rows, vocab, stride, x.data_ptr(), 0 if tok is None else tok.data_ptr(), top_n, lp.data_ptr() if "lp" in want else 0, ent.data_ptr() if "ent" in want else 0,
                             ids.data_ptr() if top_n else 0, top.data_ptr() if top_n else 0, (stream or torch.cuda.current_stream()).cuda_stream)
    torch.cuda.synchronize()
    return [a.cpu().numpy() for a in (lp, ent, ids, top)]


def _check(x, tokens, top_n, got):
    """x [rows, vocab]: finite or -infinity, in every row something finite."""
    lp, ent, ids, top = got
    y = x.double().cpu().numpy()
    for r in range(y.shape[0]):
        m = y[r].max()
        with np.errstate(invalid="ignore", divide="ignore", under="ignore"):
            d = y[r] - m
            w = np.exp(d)
            s = w.sum()
            p = w / s
            live = p > 0
            spread = float((p[live] * -d[live]).sum())
            ref, H = d - np.log(s), float(np.log(s) + spread)
        e = 2.0 ** -24 * (y.shape[1] / 256 + 40 + spread)
        def near(got, i):
            if y[r, i] == -math.inf or ref[i] < -3e38:
                return got == -math.inf or got < -3e38
            return abs(float(got) - ref[i]) <= e + 2.0 ** -23 * (abs(ref[i]) + abs(d[i]))
        if tokens is not None:
            assert near(lp[r], tokens[r]), (r, lp[r], ref[tokens[r]])
        assert abs(float(ent[r]) - H) <= e * (1 + 2 * spread) + 2.0 ** -23 * H, (r, ent[r], H)
        if top_n:
            order = np.argsort(-y[r], kind="stable")[:top_n]
            assert np.array_equal(ids[r], order), (r, ids[r], order)
            assert all(near(top[r, j], i) for j, i in enumerate(order))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 33, 255, 1000, 4097, 8191, 20001, 151936])
@pytest.mark.parametrize("rows", [1, 3])
def test_sizes(dtype, vocab, rows):
    torch.manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, device="cuda") * 3).to(TYPES[dtype][1])
    tokens = [(r * 7919 + vocab // 2) % vocab for r in range(rows)]
    for n in {0, 1, min(vocab, 5), min(vocab, 32)}:
        _check(x, tokens, n, _call(x, tokens, n))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [40, 150, 400])
def test_many_rows(dtype, rows):
    """From a cluster of blocks a row to one block a row."""
    torch.manual_seed(rows)
    x = (torch.randn(rows, 9001, device="cuda") * 2).to(TYPES[dtype][1])
    tokens = torch.randint(9001, (rows,)).tolist()
    _check(x, tokens, 20, _call(x, tokens, 20))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab, stride, first", [(1001, 1003, 1), (50257, 50261, 3), (129, 200, 5)])
def test_strides_and_alignment(dtype, vocab, stride, first):
    """Rows that begin at every element, in a wider array whose other values are NaN."""
    torch.manual_seed(vocab)
    flat = torch.full((9 * stride + first,), math.nan, device="cuda", dtype=TYPES[dtype][1])
    x = flat[first:first + 9 * stride].view(9, stride)
    x[:, :vocab] = torch.randn(9, vocab, device="cuda").to(flat.dtype)
    x[-1, vocab:] = math.nan
    tokens = list(range(9))
    _check(x[:, :vocab], tokens, 6, _call(x, tokens, 6, vocab, stride))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_equal_values_ascending_and_descending(dtype):
    """Ties go to the lower id, whatever the order in which values come."""
    dt, V = TYPES[dtype][1], 30001
    i = torch.arange(V, device="cuda")
    x = torch.stack([torch.zeros(V, device="cuda"), (i % 7).float(), i.float() / 1000, (V - i).float() / 1000, torch.where(i % 2 == 0, 0.0, -0.0), (i // 3000).float()]).to(dt)
    _check(x, [0, 29999, 5, 6, 7, 8], 32, _call(x, [0, 29999, 5, 6, 7, 8], 32))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_masks(dtype):
    """-infinity, the type's lowest and largest values; fewer values left than alternatives are asked for."""
    dt = TYPES[dtype][1]
    torch.manual_seed(3)
    low = torch.finfo(dt).min
    x = torch.randn(8, 5000, device="cuda").to(dt)
    x[0, 10:] = -math.inf
    x[1, :4990] = -math.inf
    x[2, 1::2] = low
    x[3] = low
    x[4, 7] = torch.finfo(dt).max
    x[5, ::3] = low
    x[5, 1::3] = torch.finfo(dt).max
    x[6, 100:] = -math.inf
    x[6, :99] = low
    x[7, 1:] = -math.inf
    tokens = [3, 4995, 1, 0, 7, 1, 99, 0]
    _check(x, tokens, 12, _call(x, tokens, 12))
    lp = _call(x, [4000, 0, 0, 0, 0, 0, 4000, 1], 0)[0]
    assert lp[0] == lp[1] == lp[6] == lp[7] == -math.inf


@pytest.mark.parametrize("vocab", [600, 40000])
def test_rows_of_nothing_and_rows_that_are_no_numbers(vocab):
    x = torch.randn(6, vocab, device="cuda")
    clean = x.clone()
    x[1] = -math.inf
    x[2, vocab - 1] = math.nan
    x[3, 5] = math.inf
    x[4] = math.nan
    lp, ent, ids, top = _call(x, [0] * 6, 4)
    assert lp[1] == -math.inf and ent[1] == 0 and ids[1].tolist() == [0, 1, 2, 3] and (top[1] == -math.inf).all()
    for r in (2, 3, 4):
        assert np.isnan(lp[r]) and np.isnan(ent[r]) and (ids[r] == -1).all() and np.isnan(top[r]).all()
    _check(clean[[0, 5]], [0, 0], 4, [a[[0, 5]] for a in (lp, ent, ids, top)])


def test_tokens_that_are_none():
    x = torch.randn(4, 100, device="cuda")
    lp = _call(x, [5, -1, 99, -1], 0)[0]
    assert np.isnan(lp[[1, 3]]).all() and np.isfinite(lp[[0, 2]]).all()
    rc.device_status()
    lp = _call(x, [5, 100, -2, 0x7fffffff], 0)[0]
    assert np.isnan(lp[1:]).all()
    with pytest.raises(rc.RedcudaError, match="token id"):
        rc.device_status()


def test_outputs_left_out():
    x = torch.randn(3, 1000, device="cuda")
    full = _call(x, [1, 2, 3], 4)
    for want, tokens, n in ((("lp",), [1, 2, 3], 0), (("ent",), None, 0), ((), None, 4)):
        lp, ent, ids, top = _call(x, tokens, n, want=want)
        assert np.array_equal(lp, full[0]) if "lp" in want else (lp == 7).all()
        assert np.array_equal(ent, full[1]) if "ent" in want else (ent == 7).all()
        assert not n or (np.array_equal(ids, full[2]) and np.array_equal(top, full[3]))


def test_capture_and_host_form():
    x = torch.randn(5, 12345, device="cuda")
    tokens = torch.tensor([1, 2, 3, 4, 5], dtype=torch.int32, device="cuda")
    lp, ids, top = torch.zeros(5, device="cuda"), torch.zeros(5, 3, dtype=torch.int32, device="cuda"), torch.zeros(5, 3, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            rc.token_logprobs_device(0, 5, 12345, 0, x.data_ptr(), tokens.data_ptr(), 3, lp.data_ptr(), 0, ids.data_ptr(), top.data_ptr(), s.cuda_stream)
        for seed in range(3):
            torch.manual_seed(seed)
            x.copy_(torch.randn(5, 12345, device="cuda"))
            graph.replay()
            s.synchronize()
            h = rc.token_logprobs(x.cpu().numpy(), [1, 2, 3, 4, 5], 3)
            assert np.array_equal(h[0], lp.cpu().numpy()) and np.array_equal(h[2], ids.cpu().numpy()) and np.array_equal(h[3], top.cpu().numpy())
            _check(x, [1, 2, 3, 4, 5], 3, h)
    del graph
    with pytest.raises(rc.RedcudaError, match="token id"):
        rc.token_logprobs(x.cpu().numpy(), [1, 2, 3, 4, 12345])


def test_rows_beyond_32_bits():
    """Rows whose elements are counted past 2^32."""
    rows, vocab, stride = 3, 5000, (1 << 31) + 8
    if torch.cuda.mem_get_info()[0] < 20e9:
        pytest.skip("not enough memory")
    flat = torch.empty(2 * stride + vocab, dtype=torch.float16, device="cuda")
    for r in range(rows):
        flat[r * stride:r * stride + vocab] = torch.randn(vocab, device="cuda").half()
    x = torch.stack([flat[r * stride:r * stride + vocab] for r in range(rows)])
    lp, ent, ids, top = (torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(rows, 4, dtype=torch.int32, device="cuda"), torch.zeros(rows, 4, device="cuda"))
    tokens = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    rc.token_logprobs_device(1, rows, vocab, stride, flat.data_ptr(), tokens.data_ptr(), 4, lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), top.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    _check(x, [0, 1, 2], 4, [a.cpu().numpy() for a in (lp, ent, ids, top)])


@pytest.mark.parametrize("dtype, rows, vocab, top_n", [("bf16", 16, 151936, 5), ("f32", 3, 151936, 20), ("f16", 40, 50257, 32), ("bf16", 300, 20001, 1)])
def test_again_and_again(dtype, rows, vocab, top_n):
    """The same answer to the bit, every time: what a warp knows of the others' values is a matter of time and may not show."""
    x = (torch.randn(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda") * 2).to(TYPES[dtype][1])
    tokens = [(r * 977) % vocab for r in range(rows)]
    first = _call(x, tokens, top_n)
    _check(x, tokens, top_n, first)
    for _ in range(100):
        assert all(np.array_equal(a, b) for a, b in zip(first, _call(x, tokens, top_n)))
