"""The operators of a batched server as they are used together: a model of two layers (a DeltaNet layer, an attention layer) serves several sequences, their prompts at once and then token by token, all
captured decoding steps replayed from one graph; held against every sequence by itself, in 64 bits."""
import math

import numpy as np
import pytest
import torch

import dwarfstar_red_lite_b200 as rc

pytestmark = pytest.mark.gpu

GROUPS, RANK, S, N_Q, N_KV, HD, VOCAB, HIDDEN, PAGE = 2, 4, 128, 8, 2, 64, 777, 192, 16
WIDTH = 2 * GROUPS * S + RANK * S                       # a DeltaNet row: q, k, v
ATT = (N_Q + 2 * N_KV) * HD                             # an attention row: q, k, v


class Server:
    def __init__(self, seqs, positions, seed, kv="f16"):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda") / math.sqrt(s[-1])  # noqa: E731
        self.emb, self.w_dn, self.w_ba, self.w_o1 = rnd(VOCAB, HIDDEN) * 10, rnd(WIDTH, HIDDEN), rnd(2 * RANK, HIDDEN), rnd(HIDDEN, RANK * S) * 3
        self.w_at, self.w_o2, self.head = rnd(ATT, HIDDEN) * 2, rnd(HIDDEN, N_Q * HD) * 3, rnd(VOCAB, HIDDEN) * 4
        width = -(-positions // PAGE)
        n_pages = seqs * width + 2
        dt, self.type = (torch.float16, 1) if kv == "f16" else (torch.float32, 0)
        self.k, self.v = (torch.full((n_pages, PAGE, N_KV, HD), math.nan, dtype=dt, device="cuda") for _ in range(2))
        self.table = torch.randperm(n_pages, generator=g, device="cuda")[:seqs * width].int().view(seqs, width)
        self.kv = rc.PagedKv(self.type, N_KV, HD, PAGE, n_pages, self.k.data_ptr(), self.v.data_ptr())
        self.state = torch.zeros(seqs + 1, RANK, S, S, device="cuda")
        self.slots = torch.randperm(seqs + 1, generator=g, device="cuda")[:seqs].int()
        self.work = torch.empty(self.kv.attend_workspace(N_Q), dtype=torch.uint8, device="cuda")
        self.seqs = seqs

    def rows(self, x):
        """What the projections leave of hidden rows: DeltaNet rows (keys and queries of length one), gates, betas; in the type of x."""
        y = x @ self.w_dn.to(x.dtype).T
        unit = lambda z: z / z.norm(dim=-1, keepdim=True)  # noqa: E731
        q, k = unit(y[:, :GROUPS * S].reshape(-1, GROUPS, S)), unit(y[:, GROUPS * S:2 * GROUPS * S].reshape(-1, GROUPS, S))
        ba = x @ self.w_ba.to(x.dtype).T
        return torch.cat([q.flatten(1), k.flatten(1), y[:, 2 * GROUPS * S:]], 1), -torch.nn.functional.softplus(ba[:, :RANK]), torch.sigmoid(ba[:, RANK:])

    def delta(self, x, cu, stream):
        row, gate, beta = self.rows(x)
        gate, beta, out = gate.contiguous(), beta.contiguous(), torch.zeros(x.shape[0], RANK * S, device="cuda")
        dims = rc.DeltaDims(0, GROUPS, RANK, S, WIDTH, WIDTH, WIDTH)
        p = row.data_ptr()
        ptrs = (p, p + 4 * GROUPS * S, p + 8 * GROUPS * S, gate.data_ptr(), beta.data_ptr(), self.state.data_ptr(), out.data_ptr())
        if cu is None:
            rc.delta_step_device(dims, self.seqs, self.slots.data_ptr(), self.seqs + 1, *ptrs, stream)
        else:
            work = torch.empty(dims.workspace(x.shape[0], self.seqs), dtype=torch.uint8, device="cuda")
            rc.delta_rule_device(dims, x.shape[0], self.seqs, cu.data_ptr(), self.slots.data_ptr(), self.seqs + 1, *ptrs, work.data_ptr(), work.numel(), stream)
        return x + out @ self.w_o1.T

    def prefill(self, tokens, lens):
        """Prompts laid end to end; the attention of the prompt's own tokens is not needed here: only their keys and values are kept."""
        s = torch.cuda.current_stream().cuda_stream
        cu = torch.tensor(np.cumsum([0] + lens).astype(np.int32), device="cuda")
        x = self.delta(self.emb[tokens], cu, s)
        y = x @ self.w_at.T
        p, start = y.data_ptr(), torch.zeros(self.seqs, dtype=torch.int32, device="cuda")
        self.kv.append_device(self.table.data_ptr(), self.table.shape[1], self.seqs, start.data_ptr(), x.shape[0], cu.data_ptr(), 0, p + 4 * N_Q * HD, p + 4 * (N_Q + N_KV) * HD, s, ATT)
        return x

    def step(self, tokens, lens, out):
        """One token of each sequence; lens already counts it. Writes next tokens' log probabilities, entropies and alternatives."""
        s = torch.cuda.current_stream().cuda_stream
        x = self.delta(self.emb[tokens.long()], None, s)
        y = x @ self.w_at.T
        p, att = y.data_ptr(), torch.empty(self.seqs, N_Q * HD, device="cuda")
        self.kv.attend_device(self.table.data_ptr(), self.table.shape[1], self.seqs, lens.data_ptr(), N_Q, 0, p, att.data_ptr(), self.work.data_ptr(), self.work.numel(), s,
                              k_new_ptr=p + 4 * N_Q * HD, v_new_ptr=p + 4 * (N_Q + N_KV) * HD, q_stride=ATT, new_stride=ATT)
        logits = (x + att @ self.w_o2.T) @ self.head.T
        rc.token_logprobs_device(0, self.seqs, VOCAB, VOCAB, logits.data_ptr(), tokens.data_ptr(), 4, out["lp"].data_ptr(), out["ent"].data_ptr(), out["ids"].data_ptr(), out["top"].data_ptr(), s)


def _alone(sv, tokens, n_prompt, kv16):
    """The same model for one sequence in 64 bits: of every token behind the prompt, its logits."""
    x = sv.emb[tokens].double()
    row, gate, beta = sv.rows(x)
    q, k, v = row[:, :GROUPS * S].view(-1, GROUPS, S), row[:, GROUPS * S:2 * GROUPS * S].view(-1, GROUPS, S), row[:, 2 * GROUPS * S:].view(-1, RANK, S)
    m, outs = torch.zeros(RANK, S, S, dtype=torch.float64, device="cuda"), []
    for t in range(len(tokens)):
        kk, qq = k[t].repeat_interleave(RANK // GROUPS, 0), q[t].repeat_interleave(RANK // GROUPS, 0)
        m = m * torch.exp(gate[t])[:, None, None]
        d = (v[t] - torch.einsum("hij,hj->hi", m, kk)) * beta[t][:, None]
        m = m + d[:, :, None] * kk[:, None]
        outs.append(torch.einsum("hij,hj->hi", m, qq).flatten() / math.sqrt(S))
    x = x + torch.stack(outs) @ sv.w_o1.double().T
    y = x @ sv.w_at.double().T
    qa, ka, va = y[:, :N_Q * HD].view(-1, N_Q, HD), y[:, N_Q * HD:(N_Q + N_KV) * HD].view(-1, N_KV, HD), y[:, (N_Q + N_KV) * HD:].view(-1, N_KV, HD)
    if kv16:
        ka, va = ka.half().double(), va.half().double()
    ka, va = ka.repeat_interleave(N_Q // N_KV, 1), va.repeat_interleave(N_Q // N_KV, 1)
    logits = []
    for t in range(n_prompt, len(tokens)):
        w = torch.softmax(torch.einsum("hd,phd->hp", qa[t], ka[:t + 1]) / math.sqrt(HD), -1)
        logits.append((x[t] + torch.einsum("hp,phd->hd", w, va[:t + 1]).flatten() @ sv.w_o2.double().T) @ sv.head.double().T)
    return torch.stack(logits), m


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_prompts_then_captured_steps(kv):
    lens, steps = [37, 0, 150, 1, 65], 9
    torch.backends.cuda.matmul.allow_tf32 = False
    sv = Server(len(lens), 200, 5, kv)
    rng = np.random.default_rng(3)
    seqs = [rng.integers(0, VOCAB, n + steps) for n in lens]
    sv.prefill(torch.from_numpy(np.concatenate([s[:n] for s, n in zip(seqs, lens)])).cuda(), lens)
    tokens, at = torch.zeros(len(lens), dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = dict(lp=torch.zeros(len(lens), device="cuda"), ent=torch.zeros(len(lens), device="cuda"), ids=torch.zeros(len(lens), 4, dtype=torch.int32, device="cuda"),
               top=torch.zeros(len(lens), 4, device="cuda"))
    state, side, got = sv.state.clone(), torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        at += 1
        sv.step(tokens, at, out)                       # a first call ahead of the capture, undone again
        sv.state.copy_(state)
        at -= 1
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            at += 1
            sv.step(tokens, at, out)
        for i in range(steps):
            tokens.copy_(torch.tensor([s[n + i] for s, n in zip(seqs, lens)], dtype=torch.int32))
            graph.replay()
            side.synchronize()
            got.append({k: v.clone() for k, v in out.items()})
    rc.device_status()
    for b, n in enumerate(lens):
        logits, m = _alone(sv, torch.from_numpy(seqs[b]).cuda(), n, kv == "f16")
        # 32-bit layers of some hundred sums each; a key or value that lies next to a rounding border of fp16 may fall to either side: half a step of one value among N_KV HD rows
        tol = 2e-3 if kv == "f16" else 2e-4
        for i in range(steps):
            y = torch.log_softmax(logits[i], 0)
            assert abs(float(got[i]["lp"][b]) - float(y[seqs[b][n + i]])) < tol
            assert abs(float(got[i]["ent"][b]) + float((y.exp() * y).sum())) < tol
            best = torch.sort(y, descending=True)
            assert float((got[i]["top"][b].double() - best.values[:4]).abs().max()) < tol
            for j in range(4):                         # an id is the best's, or as likely as the best within the tolerance
                assert abs(float(y[int(got[i]["ids"][b, j])] - best.values[j])) < 2 * tol
        assert float((sv.state[int(sv.slots[b])].double() - m).abs().max()) < 1e-4
    del graph


def test_two_streams_at_once():
    """Two streams that each run all operators on arrays and workspaces of their own, at the same time: every answer is the one that it is alone, to the bit."""
    g = torch.Generator(device="cuda").manual_seed(21)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def setup(kv16, lens, prompt, rows):
        n, width = len(lens), -(-max(lens) // PAGE)
        dt = torch.bfloat16 if kv16 else torch.float32
        d = dict(n=n, width=width, rows=rows, k=rnd(n * width, PAGE, N_KV, HD).to(dt), v=rnd(n * width, PAGE, N_KV, HD).to(dt), type=30 if kv16 else 0,
                 table=torch.randperm(n * width, generator=g, device="cuda").int().view(n, width), lens=ints(lens), q=rnd(n, N_Q, HD).to(dt), att=torch.empty(n, N_Q, HD, device="cuda", dtype=dt))
        d["kv"] = rc.PagedKv(d["type"], N_KV, HD, PAGE, n * width, d["k"].data_ptr(), d["v"].data_ptr())
        d["work"] = torch.empty(d["kv"].attend_workspace(N_Q), dtype=torch.uint8, device="cuda")
        d["dims"] = rc.DeltaDims(d["type"], GROUPS, RANK, S)
        unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(dt)  # noqa: E731
        T = sum(prompt)
        d["T"], d["cu"], d["m"] = T, ints(np.cumsum([0] + prompt).tolist()), len(prompt)
        d["dn"] = [unit(rnd(T, GROUPS, S)), unit(rnd(T, GROUPS, S)), rnd(T, RANK, S).to(dt), -rnd(T, RANK).abs(), torch.sigmoid(rnd(T, RANK))]
        d["state0"], d["dout"] = rnd(len(prompt), RANK, S, S), torch.empty(T, RANK, S, device="cuda", dtype=dt)
        d["state"] = d["state0"].clone()
        d["dwork"] = torch.empty(d["dims"].workspace(T, d["m"]), dtype=torch.uint8, device="cuda")
        d["x"], d["tok"] = rnd(rows, 20001).to(dt), ints(list(range(rows)))
        d["lp"], d["ids"], d["top"] = torch.empty(2, rows, device="cuda"), torch.empty(rows, 4, dtype=torch.int32, device="cuda"), torch.empty(rows, 4, device="cuda")
        return d

    def run(d, s):
        d["kv"].attend_device(d["table"].data_ptr(), d["width"], d["n"], d["lens"].data_ptr(), N_Q, d["type"], d["q"].data_ptr(), d["att"].data_ptr(), d["work"].data_ptr(), d["work"].numel(), s)
        rc.delta_rule_device(d["dims"], d["T"], d["m"], d["cu"].data_ptr(), 0, d["m"], *[a.data_ptr() for a in d["dn"]], d["state"].data_ptr(), d["dout"].data_ptr(), d["dwork"].data_ptr(),
                             d["dwork"].numel(), s)
        rc.token_logprobs_device(d["type"], d["rows"], 20001, 0, d["x"].data_ptr(), d["tok"].data_ptr(), 4, d["lp"][0].data_ptr(), d["lp"][1].data_ptr(), d["ids"].data_ptr(), d["top"].data_ptr(), s)

    got = lambda d: [d[n].clone() for n in ("att", "dout", "state", "lp", "ids", "top")]  # noqa: E731
    both = [setup(True, [700, 3, 1900, 0, 64] * 9, [200, 70, 0, 333], 3), setup(False, [90, 17], [500, 1], 150)]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    alone = []
    for d, s in zip(both, streams):
        run(d, s.cuda_stream)
        torch.cuda.synchronize()
        alone.append(got(d))
        assert all(bool(a.float().isfinite().all()) for a in alone[-1])
    for _ in range(20):
        for d in both:
            d["state"].copy_(d["state0"])
            for n in ("att", "dout", "lp", "ids", "top"):
                d[n].fill_(7)
        torch.cuda.synchronize()
        for _ in range(3):                                # the second and third run go on from the states of the one before: only the outputs of the attention are the same
            for d, s in zip(both, streams):
                run(d, s.cuda_stream)
        torch.cuda.synchronize()
        for d, want in zip(both, alone):
            now = got(d)
            assert all(torch.equal(now[i], want[i]) for i in (0, 3, 4, 5))
        for d in both:
            d["state"].copy_(d["state0"])
        torch.cuda.synchronize()
        for d, s in zip(both, streams):
            run(d, s.cuda_stream)
        torch.cuda.synchronize()
        for d, want in zip(both, alone):
            assert all(torch.equal(a, b) for a, b in zip(got(d), want))
    rc.device_status()
