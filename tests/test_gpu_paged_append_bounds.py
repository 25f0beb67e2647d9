"""Rows of prompts to a paged cache under bounds of which some cannot be: those sequences are reported and left out, every other one has all of its rows in its pages. Copies and conversions, so
everything is compared to the bit."""
import numpy as np
import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu

PAGE = 8


def _run(T, cu):
    """Every sequence begins at position 1 of pages of its own; value t + 1 in row t, everything else 0. Returns K and V as [sequence][position]."""
    n = len(cu) - 1
    width = -(-(T + 2) // PAGE)
    k, v = (torch.zeros(n * width, PAGE, 1, 64, device="cuda") for _ in range(2))
    kv = rc.PagedKv(0, 1, 64, PAGE, n * width, k.data_ptr(), v.data_ptr())
    table = torch.arange(n * width, dtype=torch.int32, device="cuda")
    rows = torch.arange(1, T + 1, device="cuda", dtype=torch.float32)[:, None].expand(T, 64).contiguous()
    bounds, start = torch.tensor(cu, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda")
    neg = -rows
    torch.cuda.synchronize()
    kv.append_device(table.data_ptr(), width, n, start.data_ptr(), T, bounds.data_ptr(), 0, rows.data_ptr(), neg.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert bool((k == k[..., :1]).all()) and bool((v == v[..., :1]).all())
    return [x[..., 0, 0].reshape(n, width * PAGE).cpu().numpy() for x in (k, v)]


def _want(T, cu, served):
    n = len(cu) - 1
    want = np.zeros((n, -(-(T + 2) // PAGE) * PAGE), np.float32)
    for b in served:
        want[b, 1:1 + cu[b + 1] - cu[b]] = np.arange(cu[b] + 1, cu[b + 1] + 1)
    return want


BIG = [3 * b for b in range(101)]


@pytest.mark.parametrize("T, cu", [
    (5, [0, 999]), (5, [-1, 3]), (5, [6, 7]), (9, [0, 3, 6, 0, 0]), (9, [0, 3, 6, -1, 9]), (9, [0, 3, 6, 2, 999]), (9, [6, 9, 0, 4]), (4, [2, 4, 0, 2, 2]),
    (300, BIG[:50] + [1000000] + BIG[51:]), (300, BIG[:64] + [-7] + BIG[65:]), (300, BIG[:70] + [0] * 31), (300, [150 + x for x in BIG[:51]] + BIG[:50]),
])
def test_the_others_are_whole(T, cu):
    n = len(cu) - 1
    fine = [b for b in range(n) if 0 <= cu[b] <= cu[b + 1] <= T]
    full = [b for b in fine if cu[b] < cu[b + 1]]
    assert len(fine) < n and not any(o != b and cu[o] < cu[b + 1] and cu[b] < cu[o + 1] for o in full for b in full)
    k, v = _run(T, cu)
    with pytest.raises(rc.RedcudaError, match="bounds"):
        rc.device_status()
    assert np.array_equal(k, _want(T, cu, fine)) and np.array_equal(v, -_want(T, cu, fine))


def test_rows_that_two_claim():
    """Bounds that fall, so that two sequences have rows in common: reported; a row that one alone has is in its pages, one that both have in those of either or both."""
    cu = [0, 3, 1, 4, 4]
    k, _ = _run(4, cu)
    with pytest.raises(rc.RedcudaError, match="bounds"):
        rc.device_status()
    want = _want(4, cu, [0, 2, 3])
    assert k[0, 1] == 1 and k[2, 3] == 4                  # rows 0 and 3
    assert bool(((k == want) | (k == 0)).all())
    assert k[0, 2] == 2 or k[2, 1] == 2
    assert k[0, 3] == 3 or k[2, 2] == 3


@pytest.mark.parametrize("T, cu", [(7, [0, 0, 3, 3, 5]), (7, [2, 4, 4, 6]), (5, [0, 5]), (1, [0, 0, 1]), (400, [2 * b for b in range(151)])])
def test_bounds_that_are_right(T, cu):
    """Rows ahead of the first sequence and behind the last are no sequence's, empty sequences have none: nothing to report."""
    k, v = _run(T, cu)
    rc.device_status()
    served = range(len(cu) - 1)
    assert np.array_equal(k, _want(T, cu, served)) and np.array_equal(v, -_want(T, cu, served))


@pytest.mark.parametrize("n", [1, 33, 1100])
def test_more_sequences_than_rows(n):
    """All but the last one empty, one bound of them beyond the rows."""
    cu = [0] * n + [2]
    k, _ = _run(3, cu)
    rc.device_status()
    assert np.array_equal(k, _want(3, cu, range(n)))
    if n > 1:
        cu[n // 2] = 4
        k, _ = _run(3, cu)
        with pytest.raises(rc.RedcudaError, match="bounds"):
            rc.device_status()
        fine = [b for b in range(n) if 0 <= cu[b] <= cu[b + 1] <= 3]
        assert np.array_equal(k, _want(3, cu, fine))
