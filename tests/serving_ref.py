"""Plain 64-bit forms of the serving operators, and how far a result may be off.

The tolerance of an attention output is the sum of what the kernels round, with u
the half step of the element type (eps / 2):
  * the output: u |O|;
  * the weights: w_j (1 + d_j) with |d_j| <= u, in the sum as in the product, moves
    O by at most u / (1 - u) * sum_j w_j |V_j - O|;
  * the scores: a 32-bit sum of D products (and its scaling) is off by at most
    (D + 8) 2^-24 sum_d |q_d k_d| / sqrt(D) = E; weights and their sum then move by
    a factor within exp(+-E), so O by at most (exp(2 E) - 1) sum_j w_j |V_j - O|;
  * exp2, the rescaling and the joins in 32 bits: a few 2^-23 of the same sum;
  * fp16 weights below its normal range are off by 2^-25 each, where the largest of
    a row's chunk is 2^8: N 2^-32 max |V| for N keys.
"""
import math

import torch

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def attend(q, k, v, limits):
    """One head in 64 bits: (O, tolerance); row i sees keys below limits[i], none: 0."""
    u = torch.finfo(q.dtype).eps / 2
    dim, m = q.shape[1], k.shape[0]
    qd, kd, vd = q.double(), k.double(), v.double()
    if m == 0 or q.shape[0] == 0:
        return torch.zeros_like(qd), torch.zeros_like(qd)
    dead = torch.arange(m, device=q.device)[None, :] >= limits[:, None]
    s = torch.mm(qd, kd.t().contiguous()) / math.sqrt(dim)
    s = s.masked_fill(dead, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    w = torch.where(total > 0, w / total, torch.zeros_like(w))
    o = torch.mm(w, vd)
    # sum_j w_j |V_j - O| <= sqrt(sum_j w_j (V_j - O)^2) (Jensen; sum_j w_j = 1)
    spread = (torch.mm(w, vd * vd) - o * o).clamp(min=0).sqrt() + 1e-9
    size = torch.mm(qd.abs(), kd.abs().t().contiguous()).masked_fill(dead, 0.0).amax(-1, keepdim=True) / math.sqrt(dim)
    e = torch.expm1(2 * (dim + 8) * 2.0 ** -24 * size)
    tol = u * o.abs() + (u / (1 - u) + e + 2.0 ** -20) * (1 + u) * spread + 1e-30
    if q.dtype == torch.float16:
        tol = tol + m * 2.0 ** -32 * vd.abs().max() + 2.0 ** -25
    return o, torch.where(total > 0, tol, torch.zeros_like(tol))


def paged(q, k_cache, v_cache, table, starts, kv_lens, block, causal):
    """(O, tolerance, rows that belong to a sequence); a page outside the cache holds zeros."""
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    inside = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    heads, heads_kv, pages = q.shape[1], k_cache.shape[1], k_cache.shape[0]
    group = heads // heads_kv
    for s, kv in enumerate(kv_lens):
        a, n = starts[s], starts[s + 1] - starts[s]
        inside[a:a + n] = True
        keys = max(0, min(kv, table.shape[1] * block))
        pos = torch.arange(keys, device=q.device)
        page = table[s].long()[pos // block]
        there = (page >= 0) & (page < pages)
        page = page.clamp(0, max(pages - 1, 0))
        if causal:
            limits = (kv - n + 1 + torch.arange(n, device=q.device)).clamp(0, keys)
        else:
            limits = torch.full((n,), keys, device=q.device)
        for g in range(heads_kv):
            k, v = (torch.where(there[:, None], c[page, g, pos % block], 0) for c in (k_cache, v_cache))
            for h in range(g * group, (g + 1) * group):
                out[a:a + n, h], tol[a:a + n, h] = attend(q[a:a + n, h], k, v, limits)
    return out, tol, inside


def cross(q, k, v, lens):
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    group = q.shape[1] // k.shape[1]
    for b, m in enumerate(lens):
        limits = torch.full((q.shape[2],), m, device=q.device)
        for h in range(q.shape[1]):
            out[b, h], tol[b, h] = attend(q[b, h], k[b, h // group, :m], v[b, h // group, :m], limits)
    return out, tol


def slots(cached, new, table, free, block, max_tokens):
    """Lists in, lists out: (table, starts, kv_lens, slots, taken), token by token."""
    table = [list(row) for row in table]
    starts, kv, slot, taken = [0], [], [], 0
    for s, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        width = len(table[s])
        for b in range(min(-(-c // block), width), min(-(-(c + n) // block), width)):
            table[s][b] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(c, c + n):
            page = table[s][p // block] if p // block < width else -1
            slot.append(page * block + p % block if page >= 0 else -1)
        starts.append(starts[-1] + n)
        kv.append(c + n)
    slot = (slot + [-1] * max_tokens)[:max_tokens]
    return table, starts, kv, slot, taken


def check(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        worst = (err / tol.clamp(min=1e-30)).max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {at}: {got[tuple(at)].item()} "
                             f"against {want[tuple(at)].item()} (tolerance {tol[tuple(at)].item():.3g}, worst {worst:.3g} times)")
