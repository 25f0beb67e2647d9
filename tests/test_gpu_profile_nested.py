"""Times of kernels by the library's own events: a bracket around others is reported beside them, and brackets of two threads do not end one another."""
import threading

import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu


def _rule(T, S, stream):
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    dims = rc.DeltaDims(0, 1, 1, S)
    rows, small, out, state, cu = z(T, 1, S), z(T, 1), z(T, 1, S), z(1, 1, S, S), torch.tensor([0, T], dtype=torch.int32, device="cuda")
    work = torch.empty(max(16, dims.workspace(T, 1)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    rc.delta_rule_device(dims, T, 1, cu.data_ptr(), 0, 1, *[rows.data_ptr()] * 3, small.data_ptr(), small.data_ptr(), state.data_ptr(), out.data_ptr(), work.data_ptr(),
                         dims.workspace(T, 1), stream.cuda_stream)
    stream.synchronize()


def test_a_bracket_around_others():
    rc.redcuda.profile_enable(True)
    for _ in range(3):
        _rule(500, 128, torch.cuda.current_stream())      # in chunks: two kernels
    _rule(5, 64, torch.cuda.current_stream())             # a token at a time: one
    got = rc.redcuda.profile_report()
    rc.redcuda.profile_enable(False)
    assert {k: v[0] for k, v in got.items()} == {"delta_rule": 4, "delta_prep": 3, "delta_chunk": 3}
    assert got["delta_rule"][1] >= got["delta_prep"][1] + got["delta_chunk"][1] > 0


def test_brackets_of_two_threads():
    streams, N = [torch.cuda.Stream() for _ in range(2)], 200
    rc.redcuda.profile_enable(True)
    threads = [threading.Thread(target=lambda s=s: [_rule(500, 128, s) for _ in range(N)]) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    got = rc.redcuda.profile_report()
    rc.redcuda.profile_enable(False)
    assert {k: v[0] for k, v in got.items()} == {"delta_rule": 2 * N, "delta_prep": 2 * N, "delta_chunk": 2 * N}
