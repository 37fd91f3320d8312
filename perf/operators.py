"""Workloads of the operators that serve token sequences of different lengths:
page plans, writes into a paged key/value cache, attention of new tokens over
that cache, and attention over packed prompts.

A request has `ctx` tokens already cached and brings `new` ones.  A plan gives
every new token a place in a cache of pages (a block table row per request, a
slot per token), a write puts the new keys and values there, the paged
attention lets the new tokens attend to all cached ones, and the packed
attention does the same for prompts whose keys lie side by side in one tensor.
Query heads share key/value heads in groups.

The lengths of a case's requests follow from the case alone (`lengths` seeds
them), its tensors from the seed of `prepare`.
"""

from __future__ import annotations

import math
import random

import torch

own = False  # True: run() calls the framework's operators, False: plain torch

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MAX_FLOPS = 1.1e13        # of any case: the largest listed one's
MAX_CACHE_BYTES = 2.7e9   # keys and values of any case


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _case(kind, requests, new, ctx, lengths, page=0, heads=0, kv_heads=0, dim=0, dtype="bf16",
          causal=True, lse=False, **more):
    """new, ctx: (lowest, highest) per request, drawn log-uniformly."""
    return {"kind": kind, "requests": requests, "new_lo": new[0], "new_hi": new[1],
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "lengths": lengths, "page": page, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal, "lse": lse,
            **more}


def listed():
    return [
        # A decoding step of 64 requests: one new token each.  Latency.
        _case("plan", 64, (1, 1), (100, 16000), 1, page=16, name="plan_step"),
        # Prompts and chunks of 500 requests admitted at once, some with
        # nothing new: 0 to 400 new tokens each.
        _case("plan", 500, (0, 400), (0, 20000), 2, page=64, name="plan_chunks"),
        # The keys and values of a decoding step of 64 requests, in one layer.
        _case("write", 64, (1, 1), (100, 3000), 1, page=16, kv_heads=8, dim=128,
              name="write_step"),
        # The keys and values of a 720p video of 16 latent frames (57,600
        # tokens), 12 heads, in pages of 64 tokens.
        _case("write", 1, (57600, 57600), (0, 0), 3, page=64, kv_heads=12, dim=128, dtype="fp16",
              name="write_video"),
        # Four short conversations, one token each: a step's latency.
        _case("paged", 4, (1, 1), (200, 1500), 4, page=16, heads=32, kv_heads=8, dim=128,
              name="step_4"),
        # A decoding step of 64 requests of 1,000 to 16,000 tokens, eight
        # query heads to a key head: the cache is read at memory speed.
        _case("paged", 64, (1, 1), (1000, 16000), 5, page=16, heads=64, kv_heads=8, dim=128,
              name="step_64"),
        # Two long contexts of about 200,000 tokens, one key head per eight
        # query heads, float16: few rows, the work split along the keys.
        _case("paged", 2, (1, 1), (180001, 220001), 6, page=64, heads=16, kv_heads=2, dim=128,
              dtype="fp16", lse=True, name="step_long"),
        # Prompt chunks of eight requests behind 500 to 30,000 cached tokens.
        _case("paged", 8, (300, 700), (500, 30000), 7, page=32, heads=32, kv_heads=8, dim=128,
              name="chunk_8"),
        # One more latent frame of a video (45 x 80 tokens) that sees all
        # 57,600 tokens before it and itself, in both directions, 40 heads.
        _case("paged", 1, (3600, 3600), (54000, 54000), 8, page=256, heads=40, kv_heads=40,
              dim=128, causal=False, name="chunk_frame"),
        # Short prompts, 64-dim heads, float16, with the softmax statistics.
        _case("packed", 7, (1, 130), (0, 0), 9, heads=12, kv_heads=12, dim=64, dtype="fp16",
              lse=True, name="prompt_short"),
        # A batch of 24 prompts of 200 to 4,000 tokens.
        _case("packed", 24, (200, 4000), (0, 0), 10, heads=32, kv_heads=8, dim=128,
              name="prompt_24"),
        # One prompt as long as a 480p video of 21 latent frames (21 x 30 x 52).
        _case("packed", 1, (32760, 32760), (0, 0), 11, heads=40, kv_heads=8, dim=128,
              name="prompt_long"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: 1 to 512 requests, 0 to 32,760 new and
    0 to 200,000 cached tokens each, 1 to 64 query heads in groups of 1 to 16,
    head dims of 40 to 128, pages of 16 to 256 tokens."""
    kind = rng.choice(("plan", "write", "paged", "paged", "paged", "packed", "packed"))
    lengths = rng.randrange(1 << 30)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    page = rng.choice((16, 32, 64, 128, 256))
    dim = rng.choice((128, 128, 64, 80, 96, 40))
    kv_heads = rng.choice((1, 2, 3, 5, 8, 12))
    heads = kv_heads * rng.choice([g for g in (1, 1, 2, 4, 5, 7, 8, 16) if g * kv_heads <= 64])
    new_hi = _log_int(rng, 1, 4000)
    new = (rng.choice((0, 1, max(1, new_hi // 8))), new_hi)
    ctx_hi = _log_int(rng, 1, 100000)
    ctx = (rng.choice((0, 1, max(1, ctx_hi // 16))), ctx_hi)
    causal = rng.random() < 0.75
    lse = rng.random() < 0.3
    if kind == "plan":
        case = _case(kind, _log_int(rng, 1, 512), new, ctx, lengths, page=page)
    elif kind == "write":
        case = _case(kind, _log_int(rng, 1, 256), new, (ctx[0], min(ctx[1], 5000)), lengths,
                     page=page, kv_heads=kv_heads, dim=dim, dtype=dtype)
    elif kind == "paged":
        step = rng.random() < 0.5  # a decoding step, or chunks
        case = _case(kind, _log_int(rng, 1, 128), (1, 1) if step else new, ctx, lengths,
                     page=page, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                     causal=causal, lse=lse)
    else:
        case = _case(kind, _log_int(rng, 1, 64), (new[0], max(1, min(32760, 4 * new_hi))),
                     (0, 0) if rng.random() < 0.75 else (0, 600), lengths, heads=heads,
                     kv_heads=kv_heads, dim=dim, dtype=dtype, causal=causal, lse=lse)
    while work(case)["flops"] > MAX_FLOPS or _cache_bytes(case) > MAX_CACHE_BYTES:
        if case["requests"] > 1:
            case["requests"] = max(1, case["requests"] // 2)
        else:
            case["new_hi"], case["ctx_hi"] = max(1, case["new_hi"] // 2), case["ctx_hi"] // 2
            case["new_lo"] = min(case["new_lo"], case["new_hi"])
            case["ctx_lo"] = min(case["ctx_lo"], case["ctx_hi"])
    if not any(_lengths(case)[0]):
        case["new_lo"] = 1  # a call brings something
    return case


def _lengths(case):
    """([new tokens], [cached tokens]) of the case's requests, log-uniform
    between their bounds."""
    rng = random.Random(case["lengths"])

    def one(lo, hi):
        return lo + _log_int(rng, 1, hi - lo + 1) - 1

    new, ctx = [], []
    for _ in range(case["requests"]):
        new.append(one(case["new_lo"], case["new_hi"]))
        # From the top: most requests are long.
        ctx.append(case["ctx_hi"] + case["ctx_lo"] - one(case["ctx_lo"], case["ctx_hi"]))
    return new, ctx


def _pages(tokens, page):
    return -(-tokens // page)


def _cache_bytes(case):
    new, ctx = _lengths(case)
    return 4.0 * (sum(new) + sum(ctx)) * max(1, case["kv_heads"]) * case["dim"]


def _pairs(case):
    """Visible (query, key) pairs per head."""
    total = 0
    for n, c in zip(*_lengths(case)):
        total += n * (n + c) - (n * (n - 1) // 2 if case["causal"] else 0)
    return total


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _clustered(shape, dtype, generator, group=128):
    """Rows of 0.8 N(0,1) noise around a centroid shared by `group` rows."""
    rows = shape[0]
    out = torch.randn(shape, device="cuda", generator=generator, dtype=dtype).mul_(0.8)
    centroids = torch.randn((-(-rows // group), *shape[1:]), device="cuda", generator=generator,
                            dtype=dtype).mul_(0.6)
    whole = rows // group * group
    if whole:
        out[:whole].view(-1, group, *shape[1:]).add_(centroids[:whole // group].unsqueeze(1))
    if whole < rows:
        out[whole:].add_(centroids[-1:])
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    new, ctx = _lengths(case)
    kind, page, requests = case["kind"], case["page"], case["requests"]
    total = sum(new)
    state = {"case": case, "new": new, "ctx": ctx}

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    state["q_start"] = ints(_starts(new))
    if kind == "packed":
        keys = [n + c for n, c in zip(new, ctx)]
        state["k_start"] = ints(_starts(keys)) if any(ctx) else None
        dtype = DTYPES[case["dtype"]]
        state["q"] = _clustered((total, case["heads"], case["dim"]), dtype, g)
        # Keys and values as two views of one projection's output.
        kv = _clustered((sum(keys), 2 * case["kv_heads"], case["dim"]), dtype, g)
        state["k"], state["v"] = kv[:, :case["kv_heads"]], kv[:, case["kv_heads"]:]
        return state
    # Physical pages in random order; the table has room for a few more.
    held = [_pages(c, page) for c in ctx]
    want = [_pages(c + n, page) for c, n in zip(ctx, new)]
    width = max(want) + 2
    pages = sum(want) + 16
    order = torch.randperm(pages, device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    host_order = order.tolist() if kind != "plan" else None
    state["pages"] = pages
    if kind == "plan":
        # Pages held so far row by row, the free ones behind them.
        table = torch.full((requests, width), -1, dtype=torch.int32)
        held_order, at = order.cpu(), 0
        for r, n in enumerate(held):
            table[r, :n] = held_order[at:at + n]
            at += n
        state.update(table=table.cuda(), free=order[at:].contiguous(), cached=ints(ctx),
                     new_lens=ints(new), total=total)
        return state
    table = torch.full((requests, width), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(want):
        table[r, :n] = torch.tensor(host_order[at:at + n], dtype=torch.int32)
        at += n
    dtype = DTYPES[case["dtype"]]
    shape = (pages, page, case["kv_heads"], case["dim"])
    # A cache in use: every row holds some request's keys, old or present.
    k_cache = _clustered((pages * page, *shape[2:]), dtype, g, page).view(shape)
    v_cache = torch.randn(shape, device="cuda", generator=g, dtype=dtype)
    state.update(k_cache=k_cache, v_cache=v_cache)
    if kind == "write":
        kv = _clustered((total, 2 * case["kv_heads"], case["dim"]), dtype, g)
        state["k"], state["v"] = kv[:, :case["kv_heads"]], kv[:, case["kv_heads"]:]
        slots = []
        for r, (n, c) in enumerate(zip(new, ctx)):
            position = torch.arange(c, c + n)
            slots.append(table[r, position // page].long() * page + position % page)
        state["slots"] = (torch.cat(slots) if slots else torch.empty(0)).long().cuda()
        return state
    state.update(table=table.cuda(), kv_lens=ints([n + c for n, c in zip(new, ctx)]),
                 q=_clustered((total, case["heads"], case["dim"]), dtype, g))
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from dit_sparse_atten_amd import ops

    case = state["case"]
    kind = case["kind"]
    if kind == "plan":
        plan = ops.paged_plan(state["cached"], state["new_lens"], state["table"], state["free"],
                              case["page"], state["total"])
        return {"table": state["table"], "q_start": plan.q_start, "kv_lens": plan.kv_lens,
                "slots": plan.slots, "status": plan.status}
    if kind == "write":
        ops.paged_write(state["k"], state["v"], state["k_cache"], state["v_cache"],
                        state["slots"])
        return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if kind == "paged":
        return ops.paged_attention(state["q"], state["k_cache"], state["v_cache"],
                                   state["table"], state["kv_lens"], state["q_start"],
                                   causal=case["causal"], return_lse=case["lse"])
    return ops.packed_attention(state["q"], state["k"], state["v"], state["q_start"],
                                state["k_start"], causal=case["causal"], return_lse=case["lse"])


def _attend(q, k, v, causal):
    """Softmax attention in float32: q [n, H, D] at the last n of m positions,
    k and v [m, KH, D]; rows without a key give 0 and a statistic of -inf."""
    n, heads, dim = q.shape
    m, kv_heads = k.shape[:2]
    group = heads // kv_heads
    out = torch.zeros((n, heads, dim), device=q.device)
    lse = torch.full((heads, n), -math.inf, device=q.device)
    if n == 0 or m == 0:
        return out, lse
    keys = k.permute(1, 2, 0).float().contiguous()
    values = v.permute(1, 0, 2).float().contiguous()
    step = max(1, (1 << 28) // (heads * m))
    for r0 in range(0, n, step):
        r1 = min(n, r0 + step)
        rows = q[r0:r1].float().view(r1 - r0, kv_heads, group, dim).permute(1, 2, 0, 3)
        s = torch.matmul(rows.reshape(kv_heads, -1, dim), keys).mul_(dim ** -0.5)
        s = s.view(kv_heads, group, r1 - r0, m)
        if causal:
            last = torch.arange(r0, r1, device=q.device) + (m - n)
            s.masked_fill_(torch.arange(m, device=q.device) > last[:, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        s.sub_(top).exp_()
        total = s.sum(-1)
        o = torch.matmul(s.view(kv_heads, -1, m), values).view(kv_heads, group, r1 - r0, dim)
        o = torch.where(total[..., None] > 0, o / total[..., None], torch.zeros_like(o))
        out[r0:r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, heads, dim)
        lse[:, r0:r1] = (top[..., 0] + total.log()).reshape(heads, r1 - r0)
    return out, lse


def _requests_plain(state):
    """(rows, keys, values) of every request."""
    case = state["case"]
    q_at, k_at = _starts(state["new"]), _starts([n + c for n, c in zip(state["new"],
                                                                      state["ctx"])])
    for r, (n, c) in enumerate(zip(state["new"], state["ctx"])):
        if case["kind"] == "packed":
            yield (q_at[r], q_at[r + 1], state["k"][k_at[r]:k_at[r + 1]],
                   state["v"][k_at[r]:k_at[r + 1]])
        else:
            rows = state["table"][r, :_pages(n + c, case["page"])].long()
            shape = (-1, case["kv_heads"], case["dim"])
            yield (q_at[r], q_at[r + 1], state["k_cache"][rows].view(shape)[:n + c],
                   state["v_cache"][rows].view(shape)[:n + c])


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "plan":
        return _plan_plain(state)
    if case["kind"] == "write":
        shape = (-1, case["kv_heads"], case["dim"])
        state["k_cache"].view(shape)[state["slots"]] = state["k"]
        state["v_cache"].view(shape)[state["slots"]] = state["v"]
        return {"k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    q = state["q"]
    out = torch.empty_like(q)
    lse = torch.empty((q.shape[1], q.shape[0]), device=q.device)
    for r0, r1, k, v in _requests_plain(state):
        o, l = _attend(q[r0:r1], k, v, case["causal"])
        out[r0:r1] = o.to(q.dtype)
        lse[:, r0:r1] = l
    return (out, lse) if case["lse"] else out


def _plan_plain(state):
    page, total = state["case"]["page"], state["total"]
    cached, new = state["cached"].long(), state["new_lens"].long()
    table, free = state["table"], state["free"]
    requests, width = table.shape
    q_start = torch.cat((new.new_zeros(1), new.cumsum(0)))
    held = torch.div(cached + page - 1, page, rounding_mode="floor")
    want = torch.div(cached + new + page - 1, page, rounding_mode="floor")
    first = (want - held).cumsum(0) - (want - held)  # of the free list, per request
    column = torch.arange(width, device=table.device)
    fresh = (column >= held[:, None]) & (column < want[:, None])
    source = torch.where(fresh, first[:, None] + column - held[:, None], 0)
    table.copy_(torch.where(fresh, free[source], table))
    token = torch.arange(total, device=table.device)
    request = torch.searchsorted(q_start[1:].contiguous(), token, right=True)
    position = cached[request] + token - q_start[request]
    index = torch.div(position, page, rounding_mode="floor")
    slots = table[request, index].long() * page + position - index * page
    status = torch.stack(((want - held).sum(), new.new_zeros(()))).to(torch.int32)
    return {"table": table, "q_start": q_start.to(torch.int32),
            "kv_lens": (cached + new).to(torch.int32), "slots": slots, "status": status}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    new, ctx = _lengths(case)
    total, requests, page = sum(new), case["requests"], case["page"]
    if case["kind"] == "plan":
        fresh = sum(_pages(c + n, page) - _pages(c, page) for n, c in zip(new, ctx))
        # Lengths in, starts and lengths out, a slot per token, the page of each
        # written to the table from the free list.
        return {"bytes": 4 * (4 * requests + 1) + 8 * total + 8 * fresh + 8, "flops": 0}
    row = 2 * case["kv_heads"] * case["dim"]
    if case["kind"] == "write":
        return {"bytes": total * (4 * row + 8), "flops": 0}
    used = sum(n + c for n, c in zip(new, ctx) if n > 0)
    out = total * case["heads"] * (2 * 2 * case["dim"] + (4 if case["lse"] else 0))
    index = 4 * sum(_pages(n + c, page) for n, c in zip(new, ctx)) if page else 0
    return {"bytes": 2 * used * row + out + index + 8 * requests,
            "flops": 4.0 * case["dim"] * case["heads"] * _pairs(case)}


# ---------------------------------------------------------------------------
# The same results in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "plan":
        return _plan_exact(state)
    if case["kind"] == "write":
        return _write_exact(state)
    q = state["q"]
    total, heads, dim = q.shape
    group = heads // case["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((heads, total), -math.inf, dtype=torch.float64, device=q.device)
    row = key = 0
    for r, (n, c) in enumerate(zip(state["new"], state["ctx"])):
        m = n + c
        if case["kind"] == "packed":
            k, v = state["k"][key:key + m], state["v"][key:key + m]
        else:
            where = torch.arange(m, device=q.device)
            page = state["table"][r].long()[where // case["page"]]
            where = where % case["page"]
            k, v = state["k_cache"][page, where], state["v_cache"][page, where]
        position = torch.arange(m, device=q.device)
        step = max(1, (1 << 27) // max(1, m))
        for h in range(case["kv_heads"]):
            kt = k[:, h].double().t().contiguous()
            vh = v[:, h].double().contiguous()
            # The rows of a key head's group, token by token.
            rows = q[row:row + n, h * group:(h + 1) * group].reshape(n * group, dim)
            for r0 in range(0, n * group, step):
                r1 = min(n * group, r0 + step)
                s = (rows[r0:r1].double() * dim ** -0.5) @ kt
                token = torch.arange(r0, r1, device=q.device) // group
                head = h * group + torch.arange(r0, r1, device=q.device) % group
                if case["causal"]:
                    s = s.masked_fill(position[None] > (c + token)[:, None], -math.inf)
                total_log = torch.logsumexp(s, dim=1)
                out[row + token, head] = torch.exp(s - total_log[:, None]) @ vh
                lse[head, row + token] = total_log
        row += n
        key += m
    return (out, lse) if case["lse"] else out


def _write_exact(state):
    """Row i of the cache after the write: the token whose slot it is, or what
    it held."""
    out = {}
    slots = state["slots"]
    rows = state["case"]["page"] * state["pages"]
    token = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    token.scatter_(0, slots, torch.arange(slots.numel(), device="cuda"))
    hit = (token >= 0)[:, None, None]
    for name, source in (("k_cache", state["k"]), ("v_cache", state["v"])):
        before = state[name].reshape(rows, *source.shape[1:]).double()
        moved = source.double()[token.clamp_min(0)] if slots.numel() else before
        out[name] = torch.where(hit, moved, before).view(state[name].shape)
    return out


def _plan_exact(state):
    """The plan, request by request."""
    page = state["case"]["page"]
    table, free = state["table"].tolist(), state["free"].tolist()
    q_start, kv_lens, slots, taken = [0], [], [], 0
    for r, (n, c) in enumerate(zip(state["new"], state["ctx"])):
        for i in range(_pages(c, page), _pages(c + n, page)):
            table[r][i] = free[taken]
            taken += 1
        slots += [table[r][i // page] * page + i % page for i in range(c, c + n)]
        q_start.append(q_start[-1] + n)
        kv_lens.append(c + n)

    def ints(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device="cuda")

    return {"table": ints(table), "q_start": ints(q_start), "kv_lens": ints(kv_lens),
            "slots": ints(slots, torch.int64), "status": ints([taken, 0])}
