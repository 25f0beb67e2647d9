"""Operators of a batched server of the hybrid model: what each has to do, on which inputs, and how it is called.

Four kinds of case:

  attend    one new token of every sequence attends over a paged key-value cache; the token's own key and value are
            written to the cache by the same call (`PagedKv.attend_device`)
  append    the keys and values of prompts are written to the pages of a cache (`PagedKv.append_device`)
  delta     the gated delta rule, for whole prompts laid end to end (`delta_rule_device`) or for one token of every
            sequence of a batch (`delta_step_device`); the states are updated in place
  logprobs  log probability of a given token, entropy and the most likely alternatives of rows of logits
            (`token_logprobs_device`)

Where `own` is false the operators are computed from elementary torch operations in 32 bits. Shapes are those of the
repository's configurations (16 query heads over 2 key-value heads of 256, 16 / 32 DeltaNet heads of 128, vocabulary
151936) and generic ones beside them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}          # ggml type ids
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# the most of a drawn case: bytes of the cache in 32 bits, of appended rows and of states, tokens of prompts, logits
HEAVIEST = {"attend": 1.0e9, "append": 1.2e8, "step": 4.0e8, "chunk": 16384, "logprobs": 1.15e8}


# ---------------------------------------------------------------------------------------------------------------- cases

def _attend(name, batch, longest, shortest, cache, q, n_q=16, n_kv=2, head_dim=256, page=64):
    c = dict(kind="attend", batch=batch, longest=longest, shortest=shortest, cache=cache, q=q, n_q=n_q, n_kv=n_kv, head_dim=head_dim, page=page)
    return dict(c, name=name) if name else c


def _append(name, seqs, tokens, start, cache, rows, n_kv=2, head_dim=256, page=64):
    c = dict(kind="append", seqs=seqs, tokens=tokens, start=start, cache=cache, rows=rows, n_kv=n_kv, head_dim=head_dim, page=page)
    return dict(c, name=name) if name else c


def _chunk(name, seqs, tokens, dtype, groups=16, rank=32, d_state=128):
    c = dict(kind="delta", form="chunk", seqs=seqs, tokens=tokens, dtype=dtype, groups=groups, rank=rank, d_state=d_state)
    return dict(c, name=name) if name else c


def _step(name, seqs, dtype, groups=16, rank=32, d_state=128):
    c = dict(kind="delta", form="step", seqs=seqs, tokens=seqs, dtype=dtype, groups=groups, rank=rank, d_state=d_state)
    return dict(c, name=name) if name else c


def _logprobs(name, rows, vocab, dtype, top):
    c = dict(kind="logprobs", rows=rows, vocab=vocab, dtype=dtype, top=top)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user, a few hundred tokens into a chat: fp32 rows over the engine's fp16 cache, where latency counts
        _attend("attend: one sequence of 613", 1, 613, 613, "f16", "f32", page=16),
        # a serving batch whose sequences are of every length, one of them empty (a padded row)
        _attend("attend: 64 ragged sequences", 64, 4096, 1, "bf16", "bf16"),
        # two users with very long documents
        _attend("attend: two long documents", 2, 131072, 100000, "f16", "f32"),
        # the default fp32 cache, a head layout of a dense model
        _attend("attend: fp32 cache, heads of 128", 24, 1999, 500, "f32", "f32", n_q=32, n_kv=8, head_dim=128, page=32),
        # one prompt chunk written to the cache of one sequence
        _append("append: chunk of 500", 1, 500, 37, "f16", "f32", page=16),
        # a batch of ragged prompts, some of which continue earlier ones
        _append("append: 32 prompts", 32, 30011, 1000, "bf16", "bf16"),
        # one prompt chunk of one sequence, in fp32 as the engine computes
        _chunk("delta rule: prompt of 2000", 1, 2000, "f32"),
        # a batch of ragged prompts laid end to end
        _chunk("delta rule: 12 prompts", 12, 16384, "bf16"),
        # one user, one token
        _step("delta rule: one token", 1, "f32"),
        # a serving batch, one token of each sequence
        _step("delta rule: batch of 96", 96, "bf16"),
        # the logits of one decoding step, five alternatives
        _logprobs("logprobs: one row", 1, 151936, "f32", 5),
        # the scoring of a prompt: a log probability for every token, twenty alternatives
        _logprobs("logprobs: prompt of 777", 777, 151936, "bf16", 20),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "chunk", "step", "logprobs"])
    if kind == "attend":
        n_q, n_kv, hd = rng.choice([(16, 2, 256), (16, 2, 256), (32, 8, 128), (32, 4, 128), (8, 8, 64), (24, 2, 128), (40, 8, 128), (16, 1, 64)])
        cache, q = rng.choice([("f16", "f32"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16")])
        batch = _log_int(rng, 1, 256)
        most = HEAVIEST["attend"] / (batch * 2 * n_kv * hd * 4)
        longest = max(1, _log_int(rng, 16, max(17, min(131072, int(most)))))
        return _attend(None, batch, longest, rng.choice([1, longest, max(1, longest // 7)]), cache, q, n_q, n_kv, hd, rng.choice([16, 32, 64, 100, 128, 256]))
    if kind == "append":
        n_kv, hd = rng.choice([(2, 256), (8, 128), (1, 64), (4, 128)])
        cache, rows = rng.choice([("f16", "f32"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
        seqs = _log_int(rng, 1, 64)
        most = int(HEAVIEST["append"] / (2 * n_kv * hd * 4))
        return _append(None, seqs, _log_int(rng, seqs, min(30011, most)), _log_int(rng, 1, 5000) - 1, cache, rows, n_kv, hd, rng.choice([16, 32, 64, 100, 256]))
    if kind == "logprobs":
        vocab = rng.choice([151936, 151936, 152064, _log_int(rng, 1000, 160000)])
        dtype = rng.choice(["f32", "f16", "bf16"])
        rows = _log_int(rng, 1, 1024)
        return _logprobs(None, max(1, min(rows, int(HEAVIEST["logprobs"] / vocab))), vocab, dtype, rng.choice([1, 5, 10, 20, 32]))
    groups, rank, S = rng.choice([(16, 32, 128), (16, 32, 128), (16, 32, 128), (8, 8, 128), (4, 16, 64), (16, 16, 64), (8, 16, 128), (2, 4, 256)])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "step":
        return _step(None, _log_int(rng, 1, max(2, int(HEAVIEST["step"] / (rank * S * S * 8)))), dtype, groups, rank, S)
    seqs = _log_int(rng, 1, 16)
    return _chunk(None, seqs, _log_int(rng, max(20, seqs), HEAVIEST["chunk"]), dtype, groups, rank, S)


# -------------------------------------------------------------------------------------------------------------- prepare

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(g, n, total):
    """n whole lengths of zero and more, of all sizes, that add up to `total`, as a list; a single one is the total."""
    if n == 1:
        return [total]
    w = torch.exp(torch.rand(n, generator=g, device="cuda") * 3.0).double()
    w[n // 2] = 0.0 if n > 2 else w[n // 2]                           # a sequence of no tokens among them
    ends = torch.round(torch.cumsum(w, 0) / w.sum() * total).long().cpu().tolist()
    return [b - a for a, b in zip([0] + ends[:-1], ends)]


def _pages(g, c, positions, n_pages):
    """A pool of n_pages pages and a table of those that hold `positions` (a list) of each sequence, scattered over the pool."""
    need = [-(-p // c["page"]) for p in positions]
    width = max(1, max(need))
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape, dtype = (n_pages, c["page"], c["n_kv"], c["head_dim"]), DTYPES[c["cache"]]
    pool = lambda: torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else torch.float16).to(dtype)  # noqa: E731
    return pool(), pool(), table


def _descriptor(c, k, v):
    import dwarfstar_red_lite_b200 as rc
    return rc.PagedKv(GGML[c["cache"]], c["n_kv"], c["head_dim"], c["page"], k.shape[0], k.data_ptr(), v.data_ptr())


def _prepare_attend(c, seed):
    g, B = _generator(seed), c["batch"]
    u = torch.rand(B, generator=g, device="cuda").cpu().tolist()
    lens = [int(round(math.exp(math.log(c["shortest"]) + x * (math.log(c["longest"]) - math.log(c["shortest"]))))) for x in u]
    lens[0] = c["longest"]
    if B > 8:
        lens[B // 2] = 0                                              # a padded row of the batch
    k, v, table = _pages(g, c, lens, B * -(-c["longest"] // c["page"]) + 3)
    dt = DTYPES[c["q"]]
    rnd = lambda heads, scale: (torch.randn(B, heads, c["head_dim"], generator=g, device="cuda") * scale).to(dt)  # noqa: E731
    s = dict(case=c, k=k, v=v, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), longest=max(lens),
             q=rnd(c["n_q"], 1.5), k_new=rnd(c["n_kv"], 1.0), v_new=rnd(c["n_kv"], 1.0))
    if own:
        s["kv"] = _descriptor(c, k, v)
        s["work"] = torch.empty(s["kv"].attend_workspace(c["n_q"]), dtype=torch.uint8, device="cuda")
    return s


def _prepare_append(c, seed):
    g, n = _generator(seed), c["seqs"]
    lens = _lengths(g, n, c["tokens"])
    start = [c["start"] if i % 2 == 0 else 0 for i in range(n)]
    k, v, table = _pages(g, c, [a + l for a, l in zip(start, lens)], (c["tokens"] + n * c["start"]) // c["page"] + n + 3)
    rnd = lambda: torch.randn(c["tokens"], c["n_kv"], c["head_dim"], generator=g, device="cuda").to(DTYPES[c["rows"]])  # noqa: E731
    ends = torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0).int()
    s = dict(case=c, k=k, v=v, table=table, start=torch.tensor(start, dtype=torch.int32, device="cuda"), cu=ends, k_new=rnd(), v_new=rnd())
    if own:
        s["kv"] = _descriptor(c, k, v)
    return s


def _prepare_delta(c, seed):
    g, n, T, S, dt = _generator(seed), c["seqs"], c["tokens"], c["d_state"], DTYPES[c["dtype"]]
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    # queries and keys as a short convolution with SiLU leaves them, of unit length
    unit = lambda x: torch.nn.functional.normalize(x * torch.sigmoid(x), dim=-1).to(dt)  # noqa: E731
    lens = [1] * n if c["form"] == "step" else _lengths(g, n, T)
    slots = n + 2                                                     # the states of other sequences lie among them
    s = dict(case=c, q=unit(rnd(T, c["groups"], S)), k=unit(rnd(T, c["groups"], S)), v=rnd(T, c["rank"], S).to(dt),
             gate=-torch.exp(rnd(T, c["rank"]) * 1.2 - 2.5), beta=torch.sigmoid(rnd(T, c["rank"])),
             state=rnd(slots, c["rank"], S, S) * 0.05, slot=torch.randperm(slots, generator=g, device="cuda")[:n].int(),
             cu=torch.tensor([0] + lens, dtype=torch.int32, device="cuda").cumsum(0).int(), lens=lens)
    if own:
        import dwarfstar_red_lite_b200 as rc
        s["dims"] = rc.DeltaDims(GGML[c["dtype"]], c["groups"], c["rank"], S)
        if c["form"] == "chunk":
            s["work"] = torch.empty(s["dims"].workspace(T, n), dtype=torch.uint8, device="cuda")
    return s


def _prepare_logprobs(c, seed):
    g = _generator(seed)
    x = torch.randn(c["rows"], c["vocab"], generator=g, device="cuda")
    x *= 2.5
    tokens = torch.randint(c["vocab"], (c["rows"],), generator=g, device="cuda")
    x[torch.arange(c["rows"], device="cuda"), tokens] += 12.0         # the given token is often a likely one
    return dict(case=c, x=x.to(DTYPES[c["dtype"]]), tokens=tokens.int())


def prepare(case, seed):
    return {"attend": _prepare_attend, "append": _prepare_append, "delta": _prepare_delta, "logprobs": _prepare_logprobs}[case["kind"]](case, seed)


# -------------------------------------------------------------------------------------------------- run: the plain forms

def _row_of(s, seq, position):
    """Row of the flattened pool that holds `position` of sequence `seq`."""
    page = s["case"]["page"]
    return s["table"][seq, position // page].long() * page + position % page


def _plain_attend(s):
    c = s["case"]
    B, G, L = c["batch"], c["n_q"] // c["n_kv"], s["longest"]
    lens, rows = s["lens"].long(), s["k"].shape[0] * c["page"]
    kf, vf = s["k"].view(rows, c["n_kv"], -1), s["v"].view(rows, c["n_kv"], -1)
    seqs = torch.arange(B, device="cuda")
    some = lens > 0
    at = _row_of(s, seqs[some], lens[some] - 1)
    kf[at], vf[at] = s["k_new"][some].to(kf.dtype), s["v_new"][some].to(vf.dtype)
    pos = torch.arange(L, device="cuda")
    valid = pos[None] < lens[:, None]
    row = torch.where(valid, _row_of(s, seqs[:, None], pos[None]), 0)
    k, v = kf[row].float(), vf[row].float()                           # [B, L, n_kv, head_dim]
    q = s["q"].float().view(B, c["n_kv"], G, -1)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(c["head_dim"])
    x = torch.where(valid[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, torch.where(valid[..., None, None], v, 0.0).permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total)).view(B, c["n_q"])
    return {"out": out.view(B, c["n_q"], -1).to(s["q"].dtype), "lse": torch.where(some[:, None], lse, -math.inf), "k": s["k"], "v": s["v"]}


def _plain_append(s):
    c, cu = s["case"], s["cu"].long()
    t = torch.arange(c["tokens"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    at = _row_of(s, seq, s["start"].long()[seq] + t - cu[seq])
    rows = s["k"].shape[0] * c["page"]
    kf, vf = s["k"].view(rows, c["n_kv"], -1), s["v"].view(rows, c["n_kv"], -1)
    kf[at], vf[at] = s["k_new"].to(kf.dtype), s["v_new"].to(vf.dtype)
    return {"k": s["k"], "v": s["v"]}


def _plain_step(s):
    c, slot = s["case"], s["slot"].long()
    width = c["rank"] // c["groups"]
    q, k = (s[n].float().repeat_interleave(width, 1) for n in ("q", "k"))
    m = s["state"][slot] * torch.exp(s["gate"])[..., None, None]      # [B, rank, value row, key column]
    d = (s["v"].float() - (m * k[:, :, None]).sum(-1)) * s["beta"][..., None]
    m += d[..., None] * k[:, :, None]
    s["state"][slot] = m
    return {"out": ((m * q[:, :, None]).sum(-1) / math.sqrt(c["d_state"])).to(s["v"].dtype), "state": s["state"]}


def _plain_chunk(s, C=64):
    """Chunks of C tokens: what the tokens of a chunk correct in one another is solved for first, all chunks at once, then
    the states go from chunk to chunk."""
    c, slot, S, H = s["case"], s["slot"].long(), s["case"]["d_state"], s["case"]["rank"]
    n, N, T = len(s["lens"]), -(-max(max(s["lens"]), 1) // C), c["tokens"]
    width = H // c["groups"]
    pos = torch.arange(N * C, device="cuda")
    cu = s["cu"].long()
    valid = pos[None] < (cu[1:] - cu[:-1])[:, None]                   # [n, N * C]
    row = torch.where(valid, cu[:-1, None] + pos[None], 0)
    take = lambda x: torch.where(valid.view(n, -1, 1, *(1,) * (x.dim() - 2)), x[row].float(), 0.0).view(n, N, C, *x.shape[1:]).transpose(2, 3)  # noqa: E731
    q, k = (take(s[x]).repeat_interleave(width, 2) for x in ("q", "k"))       # [n, N, H, C, S]
    v, beta, g = take(s["v"]), take(s["beta"]), take(s["gate"])
    G = torch.cumsum(g.double(), -1)                                  # differences of long sums: 64 bits
    i = torch.arange(C, device="cuda")
    ratio = torch.exp(torch.where(i[:, None] >= i, G[..., :, None] - G[..., None, :], -math.inf)).float()     # decay from token j to token i >= j
    a = torch.where(i[:, None] > i, torch.matmul(k, k.transpose(-1, -2)) * ratio, 0.0) * beta[..., None]
    inv = torch.eye(C, device="cuda").expand_as(a).contiguous()       # of (1 + a), row by row
    for r in range(1, C):
        inv[..., r, :r] = -torch.matmul(a[..., r:r + 1, :r], inv[..., :r, :r])[..., 0, :]
    inv = inv * beta[..., None, :]
    p = torch.matmul(q, k.transpose(-1, -2)) * ratio
    del a, ratio
    dec = torch.exp(G).float()
    u, w = torch.matmul(inv, v), torch.matmul(inv, k * dec[..., None])
    q, k = q * dec[..., None], k * torch.exp(G[..., -1:] - G).float()[..., None]
    m, out = s["state"][slot], torch.empty_like(v)
    for t in range(N):
        d = u[:, t] - torch.matmul(w[:, t], m.transpose(-1, -2))
        out[:, t] = torch.matmul(q[:, t], m.transpose(-1, -2)) + torch.matmul(p[:, t], d)
        m = m * dec[:, t, :, -1, None, None] + torch.matmul(d.transpose(-1, -2), k[:, t])
    s["state"][slot] = m
    got = torch.empty_like(s["v"])
    got[row[valid]] = (out.transpose(2, 3).reshape(n, N * C, H, S)[valid] / math.sqrt(S)).to(got.dtype)
    return {"out": got, "state": s["state"]}


def _keys(x):
    """Whole numbers in the order of the values, the lower index first among equal ones."""
    b = x.float().contiguous().view(torch.int32).long()
    b = torch.where(b < 0, -(b & 0x7fffffff), b)
    return (b << 32) - torch.arange(x.shape[-1], device=x.device)


def _plain_logprobs(s):
    x = s["x"].float()
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    ids = torch.topk(_keys(s["x"]), s["case"]["top"], dim=-1).indices
    return {"logprob": (x.gather(1, s["tokens"].long()[:, None]) - m - log_total)[:, 0],
            "entropy": (log_total - ((x - m) * e).sum(-1, keepdim=True) / total)[:, 0],
            "top_ids": ids.int(), "top_logprobs": x.gather(1, ids) - m - log_total}


# --------------------------------------------------------------------------------------------- run: the framework's calls

def _own_attend(s):
    c, stream = s["case"], torch.cuda.current_stream().cuda_stream
    out, lse = torch.empty_like(s["q"]), torch.empty(c["batch"], c["n_q"], dtype=torch.float32, device="cuda")
    s["kv"].attend_device(s["table"].data_ptr(), s["table"].shape[1], c["batch"], s["lens"].data_ptr(), c["n_q"], GGML[c["q"]], s["q"].data_ptr(), out.data_ptr(),
                          s["work"].data_ptr(), s["work"].numel(), stream, k_new_ptr=s["k_new"].data_ptr(), v_new_ptr=s["v_new"].data_ptr(), lse_ptr=lse.data_ptr())
    return {"out": out, "lse": lse, "k": s["k"], "v": s["v"]}


def _own_append(s):
    c = s["case"]
    s["kv"].append_device(s["table"].data_ptr(), s["table"].shape[1], c["seqs"], s["start"].data_ptr(), c["tokens"], s["cu"].data_ptr(), GGML[c["rows"]],
                          s["k_new"].data_ptr(), s["v_new"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return {"k": s["k"], "v": s["v"]}


def _own_delta(s):
    c, out, stream = s["case"], torch.empty_like(s["v"]), torch.cuda.current_stream().cuda_stream
    import dwarfstar_red_lite_b200 as rc
    rows = (s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["gate"].data_ptr(), s["beta"].data_ptr(), s["state"].data_ptr(), out.data_ptr())
    if c["form"] == "step":
        rc.delta_step_device(s["dims"], c["seqs"], s["slot"].data_ptr(), s["state"].shape[0], *rows, stream)
    else:
        rc.delta_rule_device(s["dims"], c["tokens"], c["seqs"], s["cu"].data_ptr(), s["slot"].data_ptr(), s["state"].shape[0], *rows, s["work"].data_ptr(), s["work"].numel(), stream)
    return {"out": out, "state": s["state"]}


def _own_logprobs(s):
    import dwarfstar_red_lite_b200 as rc
    c, dev = s["case"], "cuda"
    lp, ent = torch.empty(c["rows"], device=dev), torch.empty(c["rows"], device=dev)
    ids, top = torch.empty(c["rows"], c["top"], dtype=torch.int32, device=dev), torch.empty(c["rows"], c["top"], device=dev)
    rc.token_logprobs_device(GGML[c["dtype"]], c["rows"], c["vocab"], c["vocab"], s["x"].data_ptr(), s["tokens"].data_ptr(), c["top"], lp.data_ptr(), ent.data_ptr(),
                             ids.data_ptr(), top.data_ptr(), torch.cuda.current_stream().cuda_stream)
    return {"logprob": lp, "entropy": ent, "top_ids": ids, "top_logprobs": top}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "delta": _own_delta, "logprobs": _own_logprobs}[kind](state)
    if kind == "delta":
        return _plain_step(state) if state["case"]["form"] == "step" else _plain_chunk(state)
    return {"attend": _plain_attend, "append": _plain_append, "logprobs": _plain_logprobs}[kind](state)


# ----------------------------------------------------------------------------------------------------------- work, exact

def work(case):
    c = case
    if c["kind"] == "attend":
        # the mean length of exp(uniform) lengths between the two ends, the first sequence at the longest
        lo, hi = c["shortest"], c["longest"]
        mean = hi if hi <= lo else (hi - lo) / math.log(hi / lo)
        rows = hi + (c["batch"] - 1 - (1 if c["batch"] > 8 else 0)) * mean
        row = c["n_kv"] * c["head_dim"] * SIZE[c["cache"]]
        small = c["batch"] * (SIZE[c["q"]] * 2 * c["head_dim"] * (c["n_q"] + c["n_kv"]) + 2 * row + 4 * c["n_q"])
        return {"bytes": 2.0 * rows * row + small, "flops": 4.0 * rows * c["n_q"] * c["head_dim"]}
    if c["kind"] == "append":
        n = 2.0 * c["tokens"] * c["n_kv"] * c["head_dim"]
        return {"bytes": n * (SIZE[c["rows"]] + SIZE[c["cache"]]), "flops": n}
    if c["kind"] == "logprobs":
        return {"bytes": float(c["rows"]) * (c["vocab"] * SIZE[c["dtype"]] + 12 + 8 * c["top"]), "flops": 6.0 * c["rows"] * c["vocab"]}
    state = c["rank"] * c["d_state"] ** 2
    token = 2 * c["d_state"] * (c["groups"] + c["rank"]) * SIZE[c["dtype"]] + 8 * c["rank"]
    return {"bytes": 8.0 * c["seqs"] * state + float(c["tokens"]) * token, "flops": 7.0 * c["tokens"] * state}


def _exact_attend(s):
    c = s["case"]
    k, v = s["k"].double(), s["v"].double()
    outs, lses = [], []
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            outs.append(torch.zeros(c["n_q"], c["head_dim"], dtype=torch.float64, device="cuda"))
            lses.append(torch.full((c["n_q"],), -math.inf, dtype=torch.float64, device="cuda"))
            continue
        pages = s["table"][b, :-(-n // c["page"])].long()
        last = pages[-1], (n - 1) % c["page"]
        k[last], v[last] = s["k_new"][b].to(s["k"].dtype).double(), s["v_new"][b].to(s["v"].dtype).double()
        K, V = (x[pages].reshape(-1, c["n_kv"], c["head_dim"])[:n].repeat_interleave(c["n_q"] // c["n_kv"], 1) if n < 20000 else None for x in (k, v))
        rows = []
        for h in range(c["n_q"]):
            kh = h // (c["n_q"] // c["n_kv"])
            Kh, Vh = (K[:, h], V[:, h]) if K is not None else (x[pages][:, :, kh].reshape(-1, c["head_dim"])[:n] for x in (k, v))
            x = Kh @ s["q"][b, h].double() / math.sqrt(c["head_dim"])
            w = torch.softmax(x, 0)
            rows.append((w @ Vh, torch.logsumexp(x, 0)))
        outs.append(torch.stack([r[0] for r in rows]))
        lses.append(torch.stack([r[1] for r in rows]))
    return {"out": torch.stack(outs), "lse": torch.stack(lses), "k": k, "v": v}


def _exact_append(s):
    c = s["case"]
    k, v, ends = s["k"].double(), s["v"].double(), s["cu"].tolist()
    for b in range(c["seqs"]):
        for t in range(ends[b], ends[b + 1], 64):
            n = min(64, ends[b + 1] - t)
            at = int(s["start"][b]) + t - ends[b] + torch.arange(n, device="cuda")
            page = s["table"][b].long()[torch.div(at, c["page"], rounding_mode="floor")]
            k[page, at % c["page"]] = s["k_new"][t:t + n].to(s["k"].dtype).double()
            v[page, at % c["page"]] = s["v_new"][t:t + n].to(s["v"].dtype).double()
    return {"k": k, "v": v}


def _exact_delta(s):
    """The recurrence, a token at a time, all sequences beside one another."""
    c, n = s["case"], len(s["lens"])
    order = sorted(range(n), key=lambda b: -s["lens"][b])
    begin, lens = [s["cu"].tolist()[b] for b in order], [s["lens"][b] for b in order]
    state = s["state"].double()
    m = state[s["slot"].long()[torch.tensor(order, device="cuda")]]
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
    first = torch.tensor(begin, device="cuda")
    head = torch.arange(c["rank"], device="cuda") // (c["rank"] // c["groups"])
    decay, alive = torch.exp(s["gate"].double()), n
    for t in range(max(lens)):
        while lens[alive - 1] <= t:
            alive -= 1
        at = first[:alive] + t
        k, q = s["k"][at][:, head].double(), s["q"][at][:, head].double()
        x = m[:alive] * decay[at][..., None, None]
        d = s["beta"][at][..., None].double() * (s["v"][at].double() - torch.einsum("bhij,bhj->bhi", x, k))
        m[:alive] = x + torch.einsum("bhi,bhj->bhij", d, k)
        out[at] = torch.einsum("bhij,bhj->bhi", m[:alive], q) / math.sqrt(c["d_state"])
    state[s["slot"].long()[torch.tensor(order, device="cuda")]] = m
    return {"out": out, "state": state}


def _exact_logprobs(s):
    lp, ent, top = [], [], []
    for r in range(s["x"].shape[0]):
        y = torch.log_softmax(s["x"][r].double(), 0)
        lp.append(y[int(s["tokens"][r])])
        ent.append(-(y.exp() * y).sum())
        top.append(torch.sort(y, descending=True).values[:s["case"]["top"]])
    return {"logprob": torch.stack(lp), "entropy": torch.stack(ent), "top_ids": None, "top_logprobs": torch.stack(top)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "delta": _exact_delta, "logprobs": _exact_logprobs}[case["kind"]](s)
