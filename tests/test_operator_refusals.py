"""What the operators of a batched server refuse, before anything is launched. The pointers are numbers that nobody reads: every call here is
refused, also where there is a device."""
import ctypes as C

import pytest

import dwarfstar_red_lite_b200 as rc
from dwarfstar_red_lite_b200.redcuda import PagedKvDesc

A = [0x10000000 * (i + 1) for i in range(12)]         # 16-byte aligned, far apart


def _kv(**kw):
    d = dict(type=1, n_kv=2, head_dim=64, page_size=16, n_pages=8, page_stride=0, token_stride=0, head_stride=0, k=A[0], v=A[1])
    d.update(kw)
    return PagedKvDesc(*d.values())


def _refused(call, message):
    assert not call(), message
    assert message in rc.lib().redcuda_last_error().decode(), rc.lib().redcuda_last_error().decode()


def _attend(kv=None, table=A[2], width=4, n_seqs=3, lens=A[3], n_q=8, q_type=0, q=A[4], q_stride=0, k_new=None, v_new=None, new_stride=0, scale=0.0, out=A[5], lse=A[6], work=A[7], nbytes=1 << 27):
    kv = kv or _kv()
    return rc.lib().redcuda_kv_attend_device(C.byref(kv), table, width, n_seqs, lens, n_q, q_type, q, q_stride, k_new, v_new, new_stride, scale, out, lse, work, nbytes, None)


@pytest.mark.parametrize("change, message", [
    (dict(kv=_kv(type=14)), "cache type 14"), (dict(kv=_kv(head_dim=96)), "heads of 96"), (dict(kv=_kv(k=None)), "null cache"), (dict(kv=_kv(n_kv=0)), "empty or too large"),
    (dict(kv=_kv(page_size=0)), "empty or too large"), (dict(kv=_kv(n_pages=0)), "empty or too large"), (dict(kv=_kv(v=A[1] + 8)), "not 16-byte aligned"),
    (dict(kv=_kv(page_stride=2048, token_stride=132, head_stride=64)), "cache stride 132"), (dict(kv=_kv(page_stride=2048, token_stride=128)), "cache stride 0"),
    (dict(kv=_kv(page_stride=1 << 45)), "cache"), (dict(table=None), "null or empty"), (dict(lens=None), "null or empty"), (dict(q=None), "null or empty"), (dict(out=None), "null or empty"),
    (dict(n_seqs=0), "null or empty"), (dict(width=0), "null or empty"), (dict(k_new=A[8]), "without a value"), (dict(v_new=A[8]), "without a value"), (dict(n_q=7), "7 query heads"),
    (dict(n_q=0), "0 query heads"), (dict(q_type=30), "queries of type 30"), (dict(q_type=7), "queries of type 7"), (dict(kv=_kv(type=30)), "queries of type 0"),
    (dict(kv=_kv(type=0), q_type=1), "queries of type 1"), (dict(q_stride=500), "row strides 500"), (dict(q_stride=513), "row strides 513"),
    (dict(k_new=A[8], v_new=A[9], new_stride=64), "row strides"), (dict(q=A[4] + 4), "not 16-byte aligned"), (dict(out=A[5] + 2), "not 16-byte aligned"), (dict(work=A[7] + 8), "not 16-byte aligned"),
    (dict(out=A[4] + 16), "lies inside the inputs"), (dict(k_new=A[5] - 16, v_new=A[9]), "lies inside the inputs"), (dict(scale=float("nan")), "not a number"),
    (dict(width=0x7ffffff0, kv=_kv(page_size=64)), "2^32 positions"), (dict(lens=A[3] + 2), "4-byte aligned"), (dict(table=A[2] + 1), "4-byte aligned"), (dict(lse=A[6] + 2), "4-byte aligned"),
    (dict(out=A[0] + 64), "inside the cache"), (dict(q=A[1] + 64), "inside the cache"), (dict(work=A[0] - 64), "inside the cache"), (dict(k_new=A[1], v_new=A[9]), "inside the cache"),
    (dict(lse=A[0]), "inside the cache"), (dict(lse=A[5] + 16), "overlap"), (dict(work=A[5] + 16), "overlap"),
])
def test_attend(change, message):
    _refused(lambda: _attend(**change), message)


def _append(kv=None, table=A[2], width=4, n_seqs=3, start=A[3], n_tokens=5, cu=A[4], t=0, k=A[5], v=A[6], stride=0):
    kv = kv or _kv()
    return rc.lib().redcuda_kv_append_device(C.byref(kv), table, width, n_seqs, start, n_tokens, cu, t, k, v, stride, None)


@pytest.mark.parametrize("change, message", [
    (dict(kv=_kv(type=8)), "cache type 8"), (dict(table=None), "null or empty"), (dict(start=None), "null or empty"), (dict(k=None), "null or empty"), (dict(v=None), "null or empty"),
    (dict(n_seqs=0), "null or empty"), (dict(t=12), "rows of type 12"), (dict(cu=None), "5 rows for 3 sequences"), (dict(stride=100), "row stride 100"), (dict(stride=130), "row stride 130"),
    (dict(k=A[5] + 4), "not 16-byte aligned"), (dict(n_tokens=0x7fffffff), "too many rows"), (dict(start=A[3] + 2), "4-byte aligned"), (dict(cu=A[4] + 1), "4-byte aligned"),
    (dict(k=A[0] + 16), "inside the cache"), (dict(v=A[1] + 512), "inside the cache"),
])
def test_append(change, message):
    _refused(lambda: _append(**change), message)


@pytest.mark.parametrize("change, n_q, message", [(dict(type=3), 8, "cache type 3"), (dict(), 5, "5 query heads"), (dict(head_dim=8), 8, "heads of 8")])
def test_attend_workspace(change, n_q, message):
    _refused(lambda: rc.lib().redcuda_kv_attend_workspace(C.byref(_kv(**change)), n_q), message)


def _delta(form="rule", dims=None, n_tokens=6, n_seqs=2, cu=A[0], slots=A[1], n_slots=4, q=A[2], k=A[3], v=A[4], gate=A[5], beta=A[6], state=A[7], out=A[8]):
    dims = dims or rc.DeltaDims(0, 2, 4, 64)
    if form == "step":
        return rc.lib().redcuda_delta_step_device(C.byref(dims), n_seqs, slots, n_slots, q, k, v, gate, beta, state, out, None)
    return rc.lib().redcuda_delta_rule_device(C.byref(dims), n_tokens, n_seqs, cu, slots, n_slots, q, k, v, gate, beta, state, out, A[9], 1 << 28, None)


@pytest.mark.parametrize("form", ["rule", "step"])
@pytest.mark.parametrize("change, message", [
    (dict(dims=rc.DeltaDims(14, 2, 4, 64)), "rows of type 14"), (dict(dims=rc.DeltaDims(0, 2, 4, 96)), "states of 96"), (dict(dims=rc.DeltaDims(0, 3, 4, 64)), "4 value heads over 3"),
    (dict(dims=rc.DeltaDims(0, 0, 4, 64)), "over 0 key heads"), (dict(dims=rc.DeltaDims(0, 2, 4, 64, 64)), "row strides"), (dict(dims=rc.DeltaDims(1, 2, 4, 64, 0, 132)), "row strides"),
    (dict(dims=rc.DeltaDims(0, 2, 4, 64, 0, 0, 0, float("nan"))), "not a number"), (dict(n_slots=0), "no states"), (dict(slots=None, n_slots=1), "2 sequences for 1 states"),
    (dict(q=None), "null argument"), (dict(gate=None), "null argument"), (dict(state=None), "null argument"), (dict(out=None), "null argument"), (dict(k=A[3] + 8), "not 16-byte aligned"),
    (dict(state=A[7] + 4), "not 16-byte aligned"), (dict(out=A[4]), "inside the inputs"), (dict(out=A[2] + 16), "inside the inputs"), (dict(state=A[4] + 64), "inside the inputs"),
    (dict(out=A[7] + 32), "inside the states"), (dict(n_seqs=0), "no sequences"), (dict(gate=A[5] + 2), "4-byte aligned"), (dict(slots=A[1] + 1), "4-byte aligned"),
])
def test_delta(form, change, message):
    _refused(lambda: _delta(form, **change), message)


def test_delta_rule_without_bounds_or_workspace():
    _refused(lambda: _delta("rule", cu=None), "no sequences")
    d = rc.DeltaDims(0, 16, 32, 128)
    need = d.workspace(5000, 2)
    assert need
    call = lambda work: rc.lib().redcuda_delta_rule_device(C.byref(d), 5000, 2, A[0], A[1], 4, A[2], A[3], A[4], A[5], A[6], A[7], A[11] * 4, work, need, None)  # noqa: E731
    for inside in (A[2], A[4] + 64, A[5], A[7] + 1024, A[11] * 4):
        _refused(lambda: call(inside), "the workspace overlaps")
    _refused(lambda: call(A[9] + 8), "aligned workspace")
    if need:
        _refused(lambda: rc.lib().redcuda_delta_rule_device(C.byref(d), 5000, 2, A[0], A[1], 4, A[2], A[3], A[4], A[5], A[6], A[7], A[11] * 4, A[9], need - 1, None), "workspace of")


def _logprobs(t=0, rows=4, vocab=100, stride=0, x=A[0], tokens=A[1], top=3, lp=A[2], ent=A[3], ids=A[4], tlp=A[5]):
    return rc.lib().redcuda_token_logprobs_device(t, rows, vocab, stride, x, tokens, top, lp, ent, ids, tlp, None)


@pytest.mark.parametrize("change, message", [
    (dict(t=2), "logits of type 2"), (dict(x=None), "null or empty"), (dict(vocab=0), "null or empty"), (dict(stride=99), "100 values 99 apart"), (dict(top=33), "33 alternatives"),
    (dict(vocab=2), "3 alternatives of 2"), (dict(ids=None), "alternatives need"), (dict(tlp=None), "alternatives need"), (dict(top=0), "alternatives need"),
    (dict(tokens=None), "of no token"), (dict(x=A[0] + 2), "not aligned"), (dict(t=1, x=A[0] + 1), "not aligned"), (dict(ent=A[0] + 64), "inside the logits"), (dict(ids=A[0]), "inside the logits"),
    (dict(lp=A[2] + 2), "4-byte aligned"), (dict(tokens=A[1] + 1), "4-byte aligned"),
])
def test_logprobs(change, message):
    _refused(lambda: _logprobs(**change), message)


def test_calls_that_are_right_reach_the_device():
    """The same calls without a change are refused only where there is no device (where there is one they are not made: the pointers are numbers)."""
    if rc.lib().redcuda_device_count():
        pytest.skip("a device is there")
    for call in (_attend, _append, _delta, lambda: _delta("step"), _logprobs, lambda: rc.lib().redcuda_kv_attend_workspace(C.byref(_kv()), 8)):
        _refused(call, "no usable CUDA device")


def test_python_forms_check_shapes():
    import numpy as np
    z = np.zeros
    with pytest.raises(ValueError):
        rc.delta_rule(z((3, 2, 64)), z((3, 2, 64)), z((3, 4, 32), np.float32), z((3, 4)), z((3, 4)), z((1, 4, 32, 32), np.float32))
    with pytest.raises(ValueError):
        rc.delta_rule(z((3, 2, 64)), z((3, 2, 64)), z((3, 4, 64), np.float32), z((3, 4)), z((3, 4)), z((1, 4, 64, 64)))
    with pytest.raises(ValueError):
        rc.token_logprobs(z((3, 10), np.float32), tokens=[1, 2])


@pytest.mark.parametrize("change, message", [(dict(work=A[4] + 16), "overlap"), (dict(work=A[2]), "overlap"), (dict(work=A[3]), "overlap"), (dict(out=A[3]), "overlap"), (dict(lse=A[4] + 64), "overlap"),
                                             (dict(lse=A[2] + 4), "overlap"), (dict(k_new=A[8], v_new=A[7] + 64), "overlap"), (dict(table=A[0] + 64), "inside the cache"),
                                             (dict(lens=A[1] + 64), "inside the cache")])
def test_attend_arrays_over_one_another(change, message):
    _refused(lambda: _attend(**change), message)


@pytest.mark.parametrize("change", [dict(table=A[0] + 64), dict(start=A[1]), dict(cu=A[0])])
def test_append_arrays_inside_the_cache(change):
    _refused(lambda: _append(**change), "inside the cache")


def test_delta_arrays_over_bounds_and_slots():
    for form in ("rule", "step"):
        _refused(lambda: _delta(form, out=A[1]), "inside the inputs")
        _refused(lambda: _delta(form, slots=A[7] + 64), "inside the inputs")
    _refused(lambda: _delta("rule", cu=A[8]), "inside the inputs")
    d = rc.DeltaDims(0, 16, 32, 128)
    for work in (A[0], A[1]):
        _refused(lambda: rc.lib().redcuda_delta_rule_device(C.byref(d), 5000, 2, A[0], A[1], 4, A[2], A[3], A[4], A[5], A[6], A[7], A[11] * 4, work, d.workspace(5000, 2), None), "the workspace overlaps")


@pytest.mark.parametrize("change", [dict(lp=A[1]), dict(ids=A[1] + 8), dict(ent=A[2] + 4), dict(tlp=A[4] + 16), dict(ids=A[2])])
def test_logprob_outputs_over_one_another(change):
    _refused(lambda: _logprobs(**change), "lies inside")
