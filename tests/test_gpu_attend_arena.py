"""Decode attention with a workspace that begins an arena which holds the call's other arrays too: what the call needs of it counts, not how much there is."""
import math

import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu


def test_workspace_at_the_head_of_an_arena():
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    B, n_kv, n_q, hd, page, width = 3, 2, 8, 64, 16, 200           # a table wide enough for the form that needs the workspace
    k, v = (torch.randn(B * width, page, n_kv, hd, generator=g, device="cuda").half() for _ in range(2))
    kv = rc.PagedKv(1, n_kv, hd, page, B * width, k.data_ptr(), v.data_ptr())
    need = kv.attend_workspace(n_q)
    sizes = dict(work=need, out=B * n_q * hd * 4, lse=B * n_q * 4, q=B * n_q * hd * 4, table=B * width * 4, lens=B * 4)
    at, total = {}, 0
    for name, n in sizes.items():
        at[name], total = total, total + -(-n // 16) * 16
    arena = torch.full((total,), 0xff, dtype=torch.uint8, device="cuda")
    base = arena.data_ptr()
    part = lambda name, dtype: arena[at[name]:at[name] + sizes[name]].view(dtype)  # noqa: E731
    q = torch.randn(B, n_q, hd, generator=g, device="cuda")
    lens = [3200, 0, 1777]
    part("q", torch.float32).copy_(q.view(-1))
    part("table", torch.int32).copy_(torch.arange(B * width, device="cuda"))
    part("lens", torch.int32).copy_(torch.tensor(lens))
    torch.cuda.synchronize()
    call = lambda bytes_: kv.attend_device(base + at["table"], width, B, base + at["lens"], n_q, 0, base + at["q"], base + at["out"], base, bytes_,  # noqa: E731
                                           torch.cuda.current_stream().cuda_stream, lse_ptr=base + at["lse"])
    call(total)
    torch.cuda.synchronize()
    rc.device_status()
    out, lse = part("out", torch.float32).view(B, n_q, hd), part("lse", torch.float32).view(B, n_q)
    for b, n in enumerate(lens):
        if not n:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        K, V = (x[b * width:(b + 1) * width].reshape(-1, n_kv, hd)[:n].double().repeat_interleave(n_q // n_kv, 1) for x in (k, v))
        x = torch.einsum("hd,phd->hp", q[b].double(), K) / math.sqrt(hd)
        w = torch.softmax(x, -1)
        # the bound of test_gpu_paged_attention.py, at its largest: 2^-23 (2 (16 A + 8) + N / 4 + 16) times the largest |v|
        A = float((torch.einsum("hd,phd->hp", q[b].double().abs(), K.abs()) / math.sqrt(hd)).max())
        tol = 2.0 ** -23 * (2 * (16 * A + 8) + n / 4 + 16) * float(V.abs().max()) + 2.0 ** -24 * float(V.abs().max())
        assert float((out[b].double() - torch.einsum("hp,phd->hd", w, V)).abs().max()) <= tol
    with pytest.raises(rc.RedcudaError, match="workspace of"):
        call(need - 16)


def test_arrays_inside_what_is_needed_are_refused():
    k = torch.zeros(64, 16, 2, 64, device="cuda").half()
    v = torch.zeros_like(k)
    kv = rc.PagedKv(1, 2, 64, 16, 64, k.data_ptr(), v.data_ptr())
    need = kv.attend_workspace(8)
    arena = torch.zeros(need + (1 << 20), dtype=torch.uint8, device="cuda")
    base, table, lens = arena.data_ptr(), torch.zeros(64, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 8, 64, device="cuda")
    torch.cuda.synchronize()
    with pytest.raises(rc.RedcudaError, match="overlap"):
        kv.attend_device(table.data_ptr(), 64, 1, lens.data_ptr(), 8, 0, q.data_ptr(), base + need - 16, base, arena.numel(), torch.cuda.current_stream().cuda_stream)
