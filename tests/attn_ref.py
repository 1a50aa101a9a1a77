"""Plain 64-bit forms of the Global blocks' operators and the bounds that the
device results are held to.

Bounds. With u = 2^-24, a row's scores s_j = scale q . k_j are sums of d exact
products (bf16 inputs) or of products rounded by u (f32), so |ds_j| <= (d + 4)
u scale sum_c |q_c k_jc| =: e_j, and p_j = exp(s_j - m) carries a relative
error of e_j + e_max and of the exponential's own 2^-20 at most. Probabilities
rounded to bf16 carry 2^-8 more. Sums of L terms in f32 add L u. So with
A = sum_j p_j |v_j| / sum_j p_j,
  |do| <= r_out |o| + (r_p + 2 (2 e_max + 2^-20 + L u)) A,
  |dlse| <= 2 e_max + 2^-20 + L u + 2^-22 |lse|,
r_out half a step of the output type, r_p = 2^-8 where probabilities are
rounded to bf16 and 0 where they stay in f32.
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def seen_causal(m: int, cached: int = 0, device="cpu"):
    """[m, cached + m]: row t sees keys up to cached + t."""
    return torch.arange(cached + m, device=device)[None, :] <= cached + torch.arange(m, device=device)[:, None]


def seen_tree(parents, cached: int):
    """[m, cached + m] for parents (a list); a node whose chain of parents is
    not a chain of earlier nodes down to -1 sees nothing."""
    m = len(parents)
    seen = torch.zeros(m, cached + m, dtype=torch.bool)
    for t in range(m):
        p, chain = t, []
        while p >= 0:
            chain.append(p)
            up = parents[p]
            if up < -1 or up >= p:
                chain = None
                break
            p = up
        if chain is not None:
            seen[t, :cached] = True
            seen[t, [cached + c for c in chain]] = True
    return seen


def attention(q, k, v, seen, scale=None, rounded_p=False):
    """q [m, H, d], k and v [L, H_kv, d] of any type, seen [m, L]. Returns
    (o, lse, bound of o, bound of lse) in f64; values nobody sees (or only
    other rows see) do not reach a row."""
    m, H, d = q.shape
    L, G = k.shape[0], H // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    qd, kd, vd = q.double(), k.double(), v.double()
    o = torch.zeros(m, H, d, dtype=torch.float64, device=q.device)
    lse = torch.full((m, H), -math.inf, dtype=torch.float64, device=q.device)
    ob, lb = torch.zeros_like(o), torch.zeros_like(lse)
    r_p = 2.0 ** -8 if rounded_p else 0.0
    for h in range(H):
        x = (qd[:, h] @ kd[:, h // G].T) * scale
        x = torch.where(seen, x, torch.tensor(-math.inf, dtype=x.dtype, device=x.device))
        top = x.amax(1, keepdim=True).clamp(min=-1e300) if L else x.new_zeros(m, 1)
        p = torch.exp(x - top)
        l = p.sum(1, keepdim=True)
        some = ~(l[:, 0] == 0)
        # per row, only over the keys it sees: 0 * NaN must not appear
        vals = vd[:, h // G]
        clean = torch.isfinite(vals).all(1)
        acc = p[:, clean] @ vals[clean]
        mag = p[:, clean] @ vals[clean].abs()
        for j in (~clean).nonzero()[:, 0].tolist():
            acc[seen[:, j]] += p[seen[:, j], j, None] * vals[j]
            mag[seen[:, j]] += p[seen[:, j], j, None] * vals[j].abs().nan_to_num(posinf=0)
        o[:, h] = torch.where(some[:, None], acc / l, 0)
        lse[:, h] = torch.where(some, (top + torch.log(l))[:, 0], -math.inf)
        size = torch.where(seen & torch.isfinite(x), (qd[:, h].abs() @ kd[:, h // G].abs().T) * scale, 0)
        e = (d + 4) * U * (size.amax(1, keepdim=True) if L else size.new_zeros(m, 1))
        rel = 2 * (2 * e + 2.0 ** -20 + L * U)
        ob[:, h] = HALF_STEP[q.dtype] * o[:, h].abs() + (r_p + rel) * torch.where(some[:, None], mag / l, 0)
        lb[:, h] = (rel / 2)[:, 0] + 2.0 ** -22 * lse[:, h].abs().nan_to_num(posinf=0)
    return o, lse, ob, lb


def assert_close(got, want, bound, what=""):
    """|got - want| <= bound wherever want is finite; non-finite where it is not."""
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities differ"
    off = (got - want).abs()[fine] - bound[fine]
    assert off.numel() == 0 or off.max() <= 0, \
        f"{what}: {int((off > 0).sum())} of {off.numel()} values off by up to {float(off.max()):.3e} more than the bound"


def step_tables(cached, fresh, table, held, free, page, max_tokens, cursor=0):
    """kv_step_tables on lists, request by request."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    cu, slots, now, missing, at = [0], [], [], 0, max(cursor, 0)
    for i, (c, f, h) in enumerate(zip(cached, fresh, held)):
        c, f, h = max(c, 0), max(f, 0), min(max(h, 0), width)
        wanted = -(-(c + f) // page) if f > 0 else 0
        for p in range(h, min(wanted, width)):
            if at < len(free):
                table[i][p] = free[at]
                at += 1
                h += 1
        missing += max(wanted - h, 0)
        now.append(h)
        for pos in range(c, c + f):
            block = table[i][pos // page] if pos // page < h else -1
            slots.append(block * page + pos % page if block >= 0 else -1)
        cu.append(cu[-1] + f)
    slots = (slots + [-1] * max_tokens)[:max_tokens]
    return cu, slots, table, now, at, missing
