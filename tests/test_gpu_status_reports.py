"""What kernels report is read once, and whole: several kinds of report of the same steps are in one message."""
import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu


def _step(slots):
    B = len(slots)
    rows, small, state = torch.zeros(B, 1, 32, device="cuda"), torch.zeros(B, 1, device="cuda"), torch.zeros(2, 1, 32, 32, device="cuda")
    out, sl = torch.zeros_like(rows), torch.tensor(slots, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    rc.delta_step_device(rc.DeltaDims(0, 1, 1, 32), B, sl.data_ptr(), 2, *[rows.data_ptr()] * 3, small.data_ptr(), small.data_ptr(), state.data_ptr(), out.data_ptr(),
                         torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()


def _append(cu, page):
    k, v = (torch.zeros(1, 8, 1, 64, device="cuda") for _ in range(2))
    kv = rc.PagedKv(0, 1, 64, 8, 1, k.data_ptr(), v.data_ptr())
    n = len(cu) - 1
    table, start, bounds = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([page] * n, [0] * n, cu))
    rows = torch.zeros(4, 64, device="cuda")
    torch.cuda.synchronize()
    kv.append_device(table.data_ptr(), 1, n, start.data_ptr(), 4, bounds.data_ptr(), 0, rows.data_ptr(), rows.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()


def _logprob(token):
    x, lp = torch.zeros(1, 16, device="cuda"), torch.zeros(1, device="cuda")
    tokens = torch.tensor([token], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    rc.token_logprobs_device(0, 1, 16, 0, x.data_ptr(), tokens.data_ptr(), 0, lp.data_ptr(), 0, 0, 0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()


CAUSES = {"slot": lambda: _step([1, 1]), "page": lambda: _append([0, 4], 3), "bounds": lambda: _append([0, 4, 2], 0), "token": lambda: _logprob(16)}


@pytest.mark.parametrize("kinds", [["slot"], ["page", "slot"], ["bounds", "token"], ["slot", "page", "bounds", "token"]])
def test_every_kind_is_named(kinds):
    for k in kinds:
        CAUSES[k]()
    with pytest.raises(rc.RedcudaError) as e:
        rc.device_status()
    assert [k for k in CAUSES if k in str(e.value)] == [k for k in CAUSES if k in kinds], str(e.value)
    rc.device_status()                                    # read and cleared
