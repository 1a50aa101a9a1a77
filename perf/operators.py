"""The serving operators of the trunk's Global blocks and of drafted trees, as
cases that can be measured: their plain torch forms, and the calls a user
makes of this package (own).

  tables   block tables and slot maps of one engine step, from request lengths
  append   K and V rows of the step's tokens written to a paged cache
  prompt   causal softmax attention with grouped heads over packed prompts
  tree     softmax attention of a tree of drafted tokens (or of one token per
           sequence) over a paged cache
  gdr_tree the gated delta rule over the same trees of drafted tokens

Sizes: heads and widths of this repository's own configurations (32 heads of
128 channels, 16 heads, and 2 heads of 32 channels), 512 live sequences, 64
packed prompts of U{1..8192} positions, grouped 4 query heads to a K/V head.
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # One decode step of 512 live requests: one token each.
        dict(name="tables: 512 requests, one token", op="tables", n=512, longest=8192, fresh=1, page=16, mix=1),
        # Admission of 64 whole prompts, some 262 thousand tokens.
        dict(name="tables: 64 prompts", op="tables", n=64, longest=0, fresh=8192, page=16, mix=2),
        # The same two steps' K and V rows into the cache.
        dict(name="append: 512 tokens", op="append", n=512, longest=8192, fresh=1, page=16, kv=8, d=128, dtype="bf16", mix=1),
        dict(name="append: 64 prompts", op="append", n=64, longest=0, fresh=8192, page=16, kv=8, d=128, dtype="bf16", mix=2),
        # The test model's width and type, a few short prompts: latency counts.
        dict(name="prompt: 4 short, f32", op="prompt", n=4, longest=64, kv=1, group=2, d=32, dtype="f32", mix=3),
        # Admission of 16 prompts of any length.
        dict(name="prompt: 16 packed", op="prompt", n=16, longest=8192, kv=8, group=4, d=128, dtype="bf16", mix=4),
        # One long document.
        dict(name="prompt: one of 32768", op="prompt", n=1, longest=-32768, kv=8, group=4, d=128, dtype="bf16", mix=5),
        # Decode of 512 live sequences, one token each.
        dict(name="tree: 512 live, one token", op="tree", n=512, longest=8192, nodes=1, page=16, kv=8, group=4, d=128, dtype="bf16", mix=6),
        # Verification of trees of 1 to 64 drafted tokens.
        dict(name="tree: 48 trees", op="tree", n=48, longest=8192, nodes=64, page=16, kv=8, group=4, d=128, dtype="bf16", mix=7),
        # One conversation with a long cache and a small tree.
        dict(name="tree: cache of 131072", op="tree", n=1, longest=-131072, nodes=-24, page=64, kv=8, group=4, d=128, dtype="bf16", mix=8),
        # The Local blocks' side of the same verification.
        dict(name="gdr_tree: one of 8", op="gdr_tree", n=1, nodes=-8, heads=16, d=128, dtype="bf16", mix=9),
        dict(name="gdr_tree: 32 trees", op="gdr_tree", n=32, nodes=64, heads=32, d=128, dtype="bf16", mix=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "prompt", "tree", "gdr_tree"])
    c = dict(op=op, mix=rng.randrange(1, 1 << 30))
    page = rng.choice([8, 16, 32, 64, 128])
    wide = dict(kv=rng.choice([1, 2, 4, 8]), d=rng.choice([32, 64, 128, 128, 128]), dtype="bf16")
    if rng.random() < 0.2:
        wide["dtype"] = "f32"
    group = rng.choice([1, 2, 3, 4, 6, 8])
    if op == "tables":
        c.update(n=_log(rng, 1, 1024), longest=_log(rng, 1, 8192), fresh=_log(rng, 1, 256), page=page)
    elif op == "append":
        c.update(n=_log(rng, 1, 512), longest=_log(rng, 1, 4096), fresh=_log(rng, 1, 512), page=page, **wide)
    elif op == "prompt":
        n, longest = _log(rng, 1, 64), _log(rng, 1, 4096)
        if wide["dtype"] == "f32" or wide["d"] == 32:
            n, longest = min(n, 8), min(longest, 1024)
        c.update(n=n, longest=longest, group=group, **wide)
    elif op == "tree":
        n, longest = _log(rng, 1, 256), _log(rng, 16, 8192)
        if wide["dtype"] == "f32":
            n = min(n, 32)
        c.update(n=n, longest=longest, nodes=_log(rng, 1, 64), page=page, group=group, **wide)
    else:
        c.update(n=_log(rng, 1, 32), nodes=_log(rng, 1, 64), heads=rng.choice([2, 8, 16, 32]),
                 d=rng.choice([32, 64, 128, 128]), dtype=wide["dtype"])
    return c


def _span(r, most, least=1):
    """A length of U{least..most}; a negative `most` is taken as it stands."""
    return -most if most < 0 else r.randint(least, max(least, most))


def _lengths(case):
    """(positions in the cache, tokens of this step) of every request: host
    numbers that belong to the case, as an engine's scheduler has them."""
    r = random.Random(case["mix"])
    n, op = case["n"], case["op"]
    if op in ("tables", "append"):
        cached = [_span(r, case["longest"]) if case["longest"] else 0 for _ in range(n)]
        return cached, [_span(r, case["fresh"]) for _ in range(n)]
    if op == "prompt":
        return [0] * n, [_span(r, case["longest"]) for _ in range(n)]
    cached = [_span(r, case["longest"], 0) for _ in range(n)] if op == "tree" else [0] * n
    return cached, [_span(r, case["nodes"]) for _ in range(n)]


def _parents(case, counts):
    """Parent of every drafted token within its own sequence's tree, -1 for a
    child of the last cached token: mostly deep, with some branching."""
    r = random.Random(case["mix"] + 1)
    return [[-1 if t == 0 else (t - 1 if r.random() < 0.4 else r.randint(-1, t - 1)) for t in range(m)]
            for m in counts]


# ------------------------------------------------------------------ inputs

def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cu(counts):
    at = [0]
    for m in counts:
        at.append(at[-1] + m)
    return at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    cached, fresh = _lengths(case)
    at = _cu(fresh)
    tokens = at[-1]
    s = dict(case=case, op=op, cached_host=cached, fresh_host=fresh, at=at, tokens=tokens,
             cu=_i32(at), cached=_i32(cached), fresh=_i32(fresh))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    if op in ("tables", "append", "tree"):
        page = case["page"]
        have = [-(-c // page) for c in cached]                      # pages that hold the cached positions
        want = [-(-(c + f) // page) for c, f in zip(cached, fresh)]  # and those that the step needs
        num_blocks = sum(want) + 8
        width = max(want)
        ids = torch.randperm(num_blocks, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["n"], width), -1, dtype=torch.int32, device="cuda")
        held = have if op == "tables" else want
        lengths = _i32(held)
        inside = torch.arange(width, device="cuda")[None, :] < lengths[:, None]
        table[inside] = ids[: sum(held)]
        s.update(page=page, table=table, held=lengths, free=ids[sum(held):].contiguous(), num_blocks=num_blocks)
    if op == "append":
        dt, kv, d = TYPES[case["dtype"]], case["kv"], case["d"]
        rows = torch.arange(tokens, device="cuda")
        seq = torch.searchsorted(s["cu"][1:].long(), rows, right=True)
        pos = s["cached"].long()[seq] + rows - s["cu"].long()[seq]
        slot = table[seq, pos // page].long() * page + pos % page
        # K and V come out of one fused projection: row slices of it.
        both = randn(tokens, 2, kv, d, dtype=dt)
        s.update(slot_map=slot, k=both[:, 0], v=both[:, 1],
                 k_cache=torch.zeros(num_blocks, kv, page, d, device="cuda", dtype=dt),
                 v_cache=torch.zeros(num_blocks, kv, page, d, device="cuda", dtype=dt))
    if op == "prompt":
        dt, kv, d, H = TYPES[case["dtype"]], case["kv"], case["d"], case["kv"] * case["group"]
        s.update(q=randn(tokens, H, d, dtype=dt), k=randn(tokens, kv, d, dtype=dt), v=randn(tokens, kv, d, dtype=dt))
    if op == "tree":
        dt, kv, d, H = TYPES[case["dtype"]], case["kv"], case["d"], case["kv"] * case["group"]
        parents = _parents(case, fresh)
        s.update(q=randn(tokens, H, d, dtype=dt), parents=parents, most=max(fresh),
                 parent=None if max(fresh) == 1 else _i32([p for seq in parents for p in seq]),
                 k_cache=randn(num_blocks, kv, page, d, dtype=dt), v_cache=randn(num_blocks, kv, page, d, dtype=dt))
    if op == "gdr_tree":
        dt, H, d, n = TYPES[case["dtype"]], case["heads"], case["d"], case["n"]
        parents = _parents(case, fresh)

        def unit(x):
            return (x / x.norm(dim=-1, keepdim=True)).to(dt)

        slots = torch.randperm(n + 8, generator=g, device="cuda")[:n].to(torch.int32)
        s.update(q=unit(randn(tokens, H, d)), k=unit(randn(tokens, H, d)), v=randn(tokens, H, d).to(dt),
                 alpha=torch.exp(-torch.nn.functional.softplus(randn(tokens, H) + 2)),
                 beta=torch.sigmoid(randn(tokens, H)), pool=0.02 * randn(n + 8, H, d, d), slots=slots,
                 parents=parents, parent=_i32([p for seq in parents for p in seq]), most=max(fresh))
    return s


# ------------------------------------------------------------------ one pass

def run(state):
    return _RUN[state["op"]](state)


def _run_tables(s):
    if own:
        from rhizome_b200 import ops
        cu, slot_map, held, cursor, missing = ops.kv_step_tables(s["cached"], s["fresh"], s["table"], s["held"],
                                                                 s["free"], s["page"], s["tokens"])
        return cu, slot_map, s["table"], held, cursor, missing
    cached, fresh, table, held, free, page = (s[x] for x in ("cached", "fresh", "table", "held", "free", "page"))
    n, width = table.shape
    zero = torch.zeros(1, dtype=torch.int64, device=table.device)
    total = (cached + fresh).long()
    cu = torch.cat([zero, torch.cumsum(fresh.long(), 0)])
    wanted = (total + page - 1) // page
    need = torch.where(fresh > 0, (wanted.clamp(max=width) - held).clamp(min=0), 0)
    before = torch.cat([zero, torch.cumsum(need, 0)])
    granted = torch.minimum((free.numel() - before[:-1]).clamp(min=0), need)
    missing = torch.where(fresh > 0, (wanted - held).clamp(min=0) - granted, 0).sum()
    now = held + granted
    col = torch.arange(width, device=table.device)[None, :]
    fresh_page = (col >= held[:, None]) & (col < now[:, None])
    take = (before[:-1, None] + col - held[:, None]).clamp(0, max(free.numel() - 1, 0))
    table.copy_(torch.where(fresh_page, free[take], table))
    rows = torch.arange(s["tokens"], device=table.device)
    seq = torch.searchsorted(cu[1:], rows, right=True).clamp(max=n - 1)
    pos = cached.long()[seq] + rows - cu[seq]
    block = table[seq, (pos // page).clamp(max=width - 1)].long()
    good = (rows < cu[-1]) & (pos // page < now[seq]) & (block >= 0)
    slot_map = torch.where(good, block * page + pos % page, -1)
    return (cu.int(), slot_map, table, now.int(), granted.sum().reshape(1).int(), missing.reshape(1).int())


def _run_append(s):
    if own:
        from rhizome_b200 import ops
        ops.kv_append(s["k"], s["v"], s["slot_map"], s["k_cache"], s["v_cache"])
        return s["k_cache"], s["v_cache"]
    block, row = s["slot_map"] // s["page"], s["slot_map"] % s["page"]
    s["k_cache"][block, :, row] = s["k"]
    s["v_cache"][block, :, row] = s["v"]
    return s["k_cache"], s["v_cache"]


def _plain_rows(q, k, v, seen, scale):
    """Rows q [m, H, d] over keys k, v [L, kv, d], all f32; seen [m, L]: which
    keys a row attends. Returns o [m, H, d]."""
    m, H, d = q.shape
    kv = k.shape[1]
    qg = q.reshape(m, kv, H // kv, d).permute(1, 2, 0, 3).reshape(kv, -1, d)        # [kv, group * m, d]
    x = torch.matmul(qg, k.permute(1, 2, 0)).mul_(scale).reshape(kv, H // kv, m, -1)
    x.masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(kv, -1, p.shape[-1]), v.permute(1, 0, 2)).reshape(kv, H // kv, m, d)
    return torch.where(total > 0, o / total, 0).permute(2, 0, 1, 3).reshape(m, H, d)


def _run_prompt(s):
    if own:
        from rhizome_b200 import ops
        return ops.attn_varlen_fwd(s["q"], s["k"], s["v"], s["cu"])
    q, k, v = s["q"], s["k"], s["v"]
    out = torch.empty_like(q)
    H, d = q.shape[1:]
    for a, b in zip(s["at"], s["at"][1:]):
        step = max(1, (1 << 28) // (H * max(1, b - a)))             # rows at a time: 1 GiB of scores
        kf, vf = k[a:b].float(), v[a:b].float()
        for r in range(a, b, step):
            e = min(b, r + step)
            n = e - a                                               # keys that these rows can see
            row = torch.arange(r - a, e - a, device=q.device)[:, None]
            seen = torch.arange(n, device=q.device)[None, :] <= row
            out[r:e] = _plain_rows(q[r:e].float(), kf[:n], vf[:n], seen, d ** -0.5).to(q.dtype)
    return out


def _run_tree(s):
    if own:
        from rhizome_b200 import ops
        return ops.attn_tree_fwd(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cached"], s["cu"], s["most"],
                                 parent=s["parent"])
    q, page, table = s["q"], s["page"], s["table"]
    out = torch.empty_like(q)
    for i, (a, b) in enumerate(zip(s["at"], s["at"][1:])):
        c, m = s["cached_host"][i], b - a
        pages = table[i, : -(-(c + m) // page)].long()
        k = s["k_cache"][pages].transpose(1, 2).reshape(-1, *s["k_cache"].shape[1:4:2])[: c + m].float()
        v = s["v_cache"][pages].transpose(1, 2).reshape(-1, *s["v_cache"].shape[1:4:2])[: c + m].float()
        seen = torch.ones(m, c + m, dtype=torch.bool, device=q.device)
        if s["parent"] is not None:
            seen[:, c:] = _ancestors(s["parent"][a:b], m)
        out[a:b] = _plain_rows(q[a:b].float(), k, v, seen, q.shape[-1] ** -0.5).to(q.dtype)
    return out


def _ancestors(parent, m):
    """[m, m]: whether node j is node i or an ancestor of it, by doubling the
    distance that the parent relation covers."""
    reach = torch.eye(m, device=parent.device)
    up = torch.zeros(m, m + 1, device=parent.device)
    up.scatter_(1, torch.where(parent < 0, m, parent).long()[:, None], 1.0)
    up = up[:, :m]
    for _ in range(max(1, m.bit_length())):
        reach = ((reach + up @ reach) > 0).float()
        up = ((up @ up) > 0).float()
    return reach > 0


def _run_gdr_tree(s):
    if own:
        from rhizome_b200 import ops
        return ops.gdr_tree_step(s["q"], s["k"], s["v"], s["alpha"], s["beta"], s["cu"], s["parent"], s["most"],
                                 state_pool=s["pool"], slot_idx=s["slots"])
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    n, d = s["cu"].numel() - 1, q.shape[-1]
    first, count = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    states = torch.empty(*q.shape, d, device=q.device)
    o = torch.empty_like(s["q"])
    root = s["pool"][s["slots"].long()]
    for t in range(s["most"]):                                       # the t-th node of every tree at once
        live = count > t
        rows = (first + t)[live]
        par = s["parent"][rows].long()
        S = torch.where((par < 0)[:, None, None, None], root[live], states[first[live] + par.clamp(min=0)])
        a, b = s["alpha"][rows][..., None, None], s["beta"][rows][..., None, None]
        kt, qt, vt = k[rows][:, :, None, :], q[rows][:, :, None, :], v[rows][:, :, :, None]
        S = a * (S - b * (S * kt).sum(-1, keepdim=True) * kt) + b * vt * kt
        states[rows] = S
        o[rows] = (S * qt).sum(-1).to(o.dtype)
    return o, states


_RUN = dict(tables=_run_tables, append=_run_append, prompt=_run_prompt, tree=_run_tree, gdr_tree=_run_gdr_tree)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    cached, fresh = _lengths(case)
    tokens = sum(fresh)
    if op == "tables":
        page = case["page"]
        new = sum(-(-(c + f) // page) - -(-c // page) for c, f in zip(cached, fresh))
        partly = sum(1 for c in cached if c % page)                   # a held page that the step writes into
        return dict(bytes=case["n"] * 5 * 4 + tokens * 8 + new * 8 + partly * 4, flops=0)
    size = 2 if case["dtype"] == "bf16" else 4
    d = case["d"]
    if op == "append":
        return dict(bytes=tokens * (4 * case["kv"] * d * size + 8), flops=0)
    if op == "gdr_tree":
        H = case["heads"]
        return dict(bytes=tokens * H * (4 * d * size + 8 + 4 * d * d) + case["n"] * H * 4 * d * d + 4 * tokens,
                    flops=tokens * H * 9 * d * d)
    kv, H = case["kv"], case["kv"] * case["group"]
    if op == "prompt":
        pairs = sum(m * (m + 1) // 2 for m in fresh)
        keys = tokens
    else:
        pairs = 0
        for c, parents in zip(cached, _parents(case, fresh)):
            depth = []
            for p in parents:
                depth.append(1 if p < 0 else depth[p] + 1)
            pairs += c * len(parents) + sum(depth)
        keys = sum(cached) + tokens
    return dict(bytes=2 * keys * kv * d * size + 2 * tokens * H * d * size, flops=4 * pairs * H * d)


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    op = case["op"]
    if op == "tables":
        return None                                                   # whole numbers
    s = prepare(case, seed)
    if op == "append":
        made = []
        for x in (s["k"], s["v"]):
            rows = torch.zeros(s["num_blocks"] * s["page"], *x.shape[1:], device=x.device, dtype=torch.float64)
            rows[s["slot_map"]] = x.double()
            made.append(rows.reshape(s["num_blocks"], s["page"], *x.shape[1:]).transpose(1, 2).contiguous())
        return made
    at = s["at"]
    if op == "gdr_tree":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        alpha, beta, pool = s["alpha"].double(), s["beta"].double(), s["pool"].double()
        H, d = q.shape[1:]
        eye = torch.eye(d, device=q.device, dtype=torch.float64)
        o, states = torch.empty_like(q), torch.empty(*q.shape, d, device=q.device, dtype=torch.float64)
        for i, parents in enumerate(s["parents"]):
            for t, p in enumerate(parents):
                x = at[i] + t
                S = pool[int(s["slots"][i])] if p < 0 else states[at[i] + p]
                kk = torch.einsum("hi,hj->hij", k[x], k[x])
                S = alpha[x][:, None, None] * torch.bmm(S, eye - beta[x][:, None, None] * kk)
                states[x] = S + beta[x][:, None, None] * torch.einsum("hi,hj->hij", v[x], k[x])
                o[x] = torch.einsum("hij,hj->hi", states[x], q[x])
        return o, states
    q = s["q"]
    H, d = q.shape[1:]
    out = torch.empty(q.shape, device=q.device, dtype=torch.float64)
    for i, (a, b) in enumerate(zip(at, at[1:])):
        if op == "prompt":
            k, v, c = s["k"][a:b], s["v"][a:b], 0
            tree = None
        else:
            c = s["cached_host"][i]
            pos = torch.arange(c + b - a, device=q.device)
            block = s["table"][i].long()[pos // s["page"]]
            k, v = s["k_cache"][block, :, pos % s["page"]], s["v_cache"][block, :, pos % s["page"]]
            tree = torch.zeros(b - a, b - a, dtype=torch.bool)
            for t, p in enumerate(s["parents"][i]):
                if p >= 0:
                    tree[t] = tree[p]
                tree[t, t] = True
            tree = tree.to(q.device)
        for h in range(H):
            kh, vh = k[:, h // case["group"]].double(), v[:, h // case["group"]].double()
            for r in range(a, b, 2048):
                e = min(b, r + 2048)
                last = c + e - a if tree is None else c + b - a
                x = q[r:e, h].double() @ kh[:last].T / math.sqrt(d)
                if tree is None:
                    x = x + torch.full_like(x, -math.inf).triu(c + r - a + 1)
                else:
                    x[:, c:] = x[:, c:].masked_fill(~tree[r - a:e - a], -math.inf)
                out[r:e, h] = torch.softmax(x, -1) @ vh[:last]
    return out
