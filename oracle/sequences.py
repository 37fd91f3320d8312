"""Oracles of the sequence operators in float64 on the CPU: attention of packed
sequences and over a paged cache with shared key/value heads, and the page plan
request by request."""

from __future__ import annotations

import math

import torch


def attend(q, k, v, causal=True, scale=None, present=None):
    """One sequence: q [n, H, D] at the last n of m positions, k and v [m, KH, D].

    present: bool [m], keys that take part (default all).  Returns (out
    [n, H, D], lse [H, n], weight [n, H, D], reach [H, n]) in float64: weight =
    sum_j p_j |v_j|, reach = the largest scale sum_d |q_d k_d| of the row's
    visible keys.  Keys that a row does not see have no part in its sums, whatever
    they hold."""
    n, heads, dim = q.shape
    m, kv_heads = k.shape[:2]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    weight = torch.zeros(n, heads, dim, dtype=torch.float64)
    lse = torch.full((heads, n), -math.inf, dtype=torch.float64)
    reach = torch.zeros(heads, n, dtype=torch.float64)
    present = torch.ones(m, dtype=torch.bool) if present is None else present.cpu()
    limits = [max(0, min(m, m - n + t + 1)) if causal else m for t in range(n)]
    full = len(set(limits)) == 1
    for kh in range(kv_heads):
        for rows in ([slice(0, n)] if full else [slice(t, t + 1) for t in range(n)]):
            if n == 0:
                continue
            seen = torch.nonzero(present[:limits[rows.start]])[:, 0]
            if seen.numel() == 0:
                continue
            heads_of = slice(kh * group, (kh + 1) * group)
            qs = q[rows, heads_of].reshape(-1, dim)  # rows of (token, head)
            ks, vs = k[seen, kh], v[seen, kh]
            s = scale * (qs @ ks.t().contiguous())
            total = torch.logsumexp(s, 1)
            p = torch.exp(s - total[:, None])
            count = len(range(*rows.indices(n)))
            out[rows, heads_of] = (p @ vs).view(count, group, dim)
            weight[rows, heads_of] = (p @ vs.abs()).view(count, group, dim)
            lse[heads_of, rows] = total.view(count, group).t()
            reach[heads_of, rows] = (scale * (qs.abs() @ ks.abs().t())).amax(1).view(
                count, group).t()
    return out, lse, weight, reach


def packed(q, k, v, q_lens, k_lens=None, causal=True, scale=None):
    """Sequences side by side; returns as ``attend`` over all rows."""
    parts, row, key = [], 0, 0
    for n, m in zip(q_lens, k_lens or q_lens):
        parts.append(attend(q[row:row + n], k[key:key + m], v[key:key + m], causal, scale))
        row, key = row + n, key + m
    return tuple(torch.cat([p[i] for p in parts], dim=1 if i in (1, 3) else 0) for i in range(4))


def paged(q, k_cache, v_cache, table, kv_lens, q_lens, causal=True, scale=None):
    """New tokens over the pages of a block table (a list of lists; an entry
    outside the cache: its keys take no part)."""
    pages, size = k_cache.shape[:2]
    parts, row = [], 0
    for r, (n, m) in enumerate(zip(q_lens, kv_lens)):
        index = torch.tensor([table[r][j // size] for j in range(m)], dtype=torch.int64)
        at = torch.arange(m) % size
        ok = (index >= 0) & (index < pages)
        rows = (index.clamp(0, max(0, pages - 1)).to(k_cache.device), at.to(k_cache.device))
        parts.append(attend(q[row:row + n], k_cache[rows], v_cache[rows], causal, scale, ok))
        row += n
    return tuple(torch.cat([p[i] for p in parts], dim=1 if i in (1, 3) else 0) for i in range(4))


def plan(cached, new, table, free, page_size, tokens):
    """(q_start, kv_lens, slots, status, table) of a step, request by request."""
    table = [list(row) for row in table]
    width = len(table[0]) if table else 0
    q_start, kv_lens, slots, needed, lost = [0], [], [], 0, 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        held = min(-(-c // page_size), width)
        want = min(-(-(c + n) // page_size), width)
        for i in range(held, want):
            table[r][i] = free[needed] if needed < len(free) else -1
            needed += 1
        for position in range(c, c + n):
            i = position // page_size
            page = table[r][i] if i < want else -1
            slot = page * page_size + position % page_size if page >= 0 else -1
            lost += slot < 0 or len(slots) >= tokens
            slots.append(slot)
        q_start.append(q_start[-1] + n)
        kv_lens.append(c + n)
    slots = (slots + [-1] * tokens)[:tokens]
    return q_start, kv_lens, slots, [needed, lost], table
