"""Workloads of the paged cache's rotated writes and of its 4-bit form.

A request has `ctx` tokens already cached and brings `new` ones.
 rotate:  the new keys turn with their positions on the way into a 16-bit cache,
          the values go there as they are, the new queries turn beside them.
 write4:  the same into a cache of 4-bit elements; the cache is read back as the
          values it stands for.
 read4:   listed pages of a 4-bit cache as 16-bit values (a prefix that another
          cache takes over).
 attend4: the new tokens' attention over a 4-bit cache.

A 4-bit cache is uint8 [pages, kv_heads, page_size, 32 G + 8], G = ceil(dim / 32).
The bytes of one page and head are, one after the other, the keys' codes
[page_size, 16 G], the values' codes [page_size, 16 G], the keys' scales
[page_size, 4] and the values' scales [page_size, 4].  32 neighbouring dims share a
scale byte b, which stands for 2^(b - 127) (255: the group is not a number); element
2 i of a row is the low half of its byte i.  Codes are a sign bit over the magnitudes
0, 0.5, 1, 1.5, 2, 3, 4, 6.  A group's exponent is the smallest whose 7-fold holds the
largest element (which then rounds to 6 at most); elements round to the nearest code,
ties to the even one.

The lengths of a case's requests follow from the case alone (`lengths` seeds
them), its tensors from the seed of `prepare`.
"""

from __future__ import annotations

import math
import random

import torch

own = False  # True: run() calls the framework's operators, False: plain torch

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EXPONENTS = {"bf16": (-125, 125), "fp16": (-23, 13)}  # of a group, by the type written
MAX_FLOPS = 4.3e12        # of any case: the largest listed one's
MAX_VALUES = 3.4e8        # keys and values in any cache that is written or read back
MAX_KEYS = 1.4e9          # keys and values of any attention


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _case(kind, requests, new, ctx, lengths, page, kv_heads, dim, heads=0, dtype="bf16", rot=0,
          halves=False, causal=True, lse=False, **more):
    """new, ctx: (lowest, highest) per request, drawn log-uniformly.  rot: leading dims
    that turn, in neighbouring pairs or (halves) in pairs half of them apart; 0: none."""
    return {"kind": kind, "requests": requests, "new_lo": new[0], "new_hi": new[1],
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "lengths": lengths, "page": page, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "rot": rot, "halves": halves,
            "causal": causal, "lse": lse, **more}


def listed():
    return [
        # A decoding step of 64 requests, one layer: 32 query and 8 key heads.  Latency.
        _case("rotate", 64, (1, 1), (100, 3000), 1, 16, 8, 128, heads=32, rot=128, halves=True,
              name="rotate_step"),
        # A 720p video of 16 latent frames (57,600 tokens), 12 heads.
        _case("rotate", 1, (57600, 57600), (0, 0), 2, 64, 12, 128, heads=12, rot=128,
              name="rotate_video"),
        # Prompts of 23 requests, 80-dim heads of which 32 dims turn, float16.
        _case("rotate", 23, (1, 700), (0, 900), 3, 32, 5, 80, heads=20, dtype="fp16", rot=32,
              halves=True, name="rotate_prompts"),
        # The first tokens of 64 answers: a step's keys into a small 4-bit cache.
        _case("write4", 64, (1, 1), (1, 60), 4, 16, 8, 128, heads=32, rot=128, halves=True,
              name="write4_step"),
        # The video's keys and values (12 heads) into a 4-bit cache.
        _case("write4", 1, (57600, 57600), (0, 0), 5, 64, 12, 128, rot=128, name="write4_video"),
        # A short shared prefix, float16.
        _case("read4", 1, (1, 1), (1000, 1000), 6, 16, 8, 128, dtype="fp16", name="read4_prefix"),
        # The video's keys and values out of a 4-bit cache.
        _case("read4", 1, (1, 1), (57600, 57600), 7, 64, 12, 128, name="read4_video"),
        # Four short conversations, one token each: a step's latency.
        _case("attend4", 4, (1, 1), (200, 1500), 8, 16, 8, 128, heads=32, name="step4_4"),
        # A decoding step of 64 requests of 1,000 to 16,000 tokens: the cache is read
        # at memory speed.
        _case("attend4", 64, (1, 1), (1000, 16000), 9, 16, 8, 128, heads=64, name="step4_64"),
        # Two long contexts of about 200,000 tokens, float16, with the statistics.
        _case("attend4", 2, (1, 1), (180001, 220001), 10, 64, 2, 128, heads=16, dtype="fp16",
              lse=True, name="step4_long"),
        # Prompt chunks of eight requests behind 500 to 30,000 cached tokens.
        _case("attend4", 8, (300, 700), (500, 30000), 11, 32, 8, 128, heads=32, name="chunk4_8"),
        # One more latent frame of a video (45 x 80 tokens) that sees all 57,600 tokens,
        # in both directions, 40 heads.
        _case("attend4", 1, (3600, 3600), (54000, 54000), 12, 256, 40, 128, heads=40,
              causal=False, name="chunk4_frame"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges: 1 to 128 requests, 0 to 4,000 new and 0 to
    100,000 cached tokens each, 1 to 64 query heads in groups of 1 to 16, head dims of
    40 to 128, pages of 16 to 256 tokens, all or a part of the dims turned."""
    kind = rng.choice(("rotate", "rotate", "write4", "write4", "read4", "attend4", "attend4",
                       "attend4"))
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
    rot = rng.choice((dim // 16 * 16, dim // 16 * 16, 32, 16))
    halves = rng.random() < 0.5
    if kind == "rotate":
        case = _case(kind, _log_int(rng, 1, 128), new, (ctx[0], min(ctx[1], 5000)), lengths, page,
                     kv_heads, dim, heads=heads, dtype=dtype, rot=rot, halves=halves)
    elif kind == "write4":
        case = _case(kind, _log_int(rng, 1, 64), new, (min(ctx[0], 50), min(ctx[1], 500)),
                     lengths, page, kv_heads, dim, heads=rng.choice((0, heads)), dtype=dtype,
                     rot=rot, halves=halves)
        if not case["heads"] and rng.random() < 0.5:
            case["rot"] = 0
    elif kind == "read4":
        case = _case(kind, _log_int(rng, 1, 16), (0, 1), ctx, lengths, page, kv_heads, dim,
                     dtype=dtype)
    else:
        step = rng.random() < 0.5  # a decoding step, or chunks
        case = _case(kind, _log_int(rng, 1, 128), (1, 1) if step else new, ctx, lengths, page,
                     kv_heads, dim, heads=heads, dtype=dtype, causal=rng.random() < 0.75,
                     lse=rng.random() < 0.3)
    limit = MAX_KEYS if kind == "attend4" else MAX_VALUES
    while work(case)["flops"] > MAX_FLOPS or _cache_values(case) > limit:
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


def _cache_pages(case):
    return sum(_pages(n + c, case["page"]) for n, c in zip(*_lengths(case))) + 3


def _cache_values(case):
    return 2.0 * _cache_pages(case) * case["page"] * case["kv_heads"] * case["dim"]


def _groups(case):
    return -(-case["dim"] // 32)


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


def _regions(cache, groups):
    """(keys' codes, values' codes, keys' scales, values' scales) of a 4-bit cache, views
    [pages, kv_heads, page_size, bytes]."""
    pages, heads, page, _ = cache.shape
    flat, code = cache.view(pages, heads, -1), page * 16 * groups
    cuts = (0, code, 2 * code, 2 * code + 4 * page, 2 * code + 8 * page)
    return tuple(flat[:, :, a:b].unflatten(2, (page, -1)) for a, b in zip(cuts, cuts[1:]))


def _cache4(case, pages, generator):
    """A 4-bit cache in use: every row holds some request's keys."""
    page, heads, groups = case["page"], case["kv_heads"], _groups(case)
    cache = torch.zeros((pages, heads, page, 32 * groups + 8), dtype=torch.uint8, device="cuda")
    kc, vc, ks, vs = _regions(cache, groups)
    step = max(1, (1 << 27) // (page * heads * case["dim"]))
    for p0 in range(0, pages, step):
        p1 = min(pages, p0 + step)
        shape = ((p1 - p0) * page, heads, case["dim"])
        for codes, scales, values in (
                (kc, ks, _clustered(shape, torch.float32, generator, page)),
                (vc, vs, torch.randn(shape, device="cuda", generator=generator))):
            c, s = _quantize(values, case["dtype"])
            codes[p0:p1] = c.view(p1 - p0, page, heads, -1).transpose(1, 2)
            scales[p0:p1, :, :, :groups] = s.view(p1 - p0, page, heads, -1).transpose(1, 2)
    return cache


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    new, ctx = _lengths(case)
    kind, page, requests = case["kind"], case["page"], case["requests"]
    total, dtype, dim = sum(new), DTYPES[case["dtype"]], case["dim"]
    state = {"case": case, "new": new, "ctx": ctx}

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    # Physical pages in random order; the table has room for a few more.
    want = [_pages(c + n, page) for c, n in zip(ctx, new)]
    width, pages = max(want) + 2, _cache_pages(case)
    order = torch.randperm(pages, device="cuda", generator=g).tolist()
    table, at = torch.full((requests, width), -1, dtype=torch.int32), 0
    for r, n in enumerate(want):
        table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    if kind == "rotate":
        # A cache in use, keys of an earlier time.
        shape = (pages, page, case["kv_heads"], dim)
        state["k_cache"] = _clustered((pages * page, *shape[2:]), dtype, g, page).view(shape)
        state["v_cache"] = torch.randn(shape, device="cuda", generator=g, dtype=dtype)
    else:
        state["cache"] = _cache4(case, pages, g)
    if kind == "read4":
        state["list"] = ints(order[:at])
        return state
    if kind == "attend4":
        state.update(table=table.cuda(), kv_lens=ints([n + c for n, c in zip(new, ctx)]),
                     q_start=ints(_starts(new)),
                     q=_clustered((total, case["heads"], dim), dtype, g))
        return state
    # Queries, keys and values as views of one projection's output.
    kv_heads, heads = case["kv_heads"], case["heads"]
    x = _clustered((total, heads + 2 * kv_heads, dim), dtype, g)
    state["q"] = x[:, :heads] if heads else None
    state["k"], state["v"] = x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    position = torch.cat([torch.arange(c, c + n) for n, c in zip(new, ctx)])
    row = torch.repeat_interleave(torch.arange(requests), torch.tensor(new))
    slots = table[row, position // page].long() * page + position % page
    state["slots"] = slots.cuda()
    state["positions"] = position.int().cuda() if case["rot"] else None
    state["cos_sin"] = None
    if case["rot"]:
        # (cos, sin) of every position's angles, from 64 bits.
        longest = max(n + c for n, c in zip(new, ctx))
        rate = 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        angle = torch.arange(longest, dtype=torch.float64, device="cuda")[:, None] * rate.cuda()
        state["cos_sin"] = torch.stack((angle.cos(), angle.sin()), -1).float()
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
    if kind == "rotate":
        q = ops.paged_write_rotary(state["k"], state["v"], state["k_cache"], state["v_cache"],
                                   state["slots"], state["positions"], state["cos_sin"],
                                   q=state["q"], halves=case["halves"])
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    if kind == "write4":
        q = ops.paged_write_fp4(state["k"], state["v"], state["cache"], state["slots"],
                                state["positions"], state["cos_sin"], q=state["q"],
                                halves=case["halves"])
        k, v = ops.paged_read_fp4(state["cache"], case["dim"], dtype=DTYPES[case["dtype"]])
        return {"q": q, "k": k, "v": v}
    if kind == "read4":
        k, v = ops.paged_read_fp4(state["cache"], case["dim"], state["list"],
                                  dtype=DTYPES[case["dtype"]])
        return {"k": k, "v": v}
    return ops.paged_attention_fp4(state["q"], state["cache"], state["table"], state["kv_lens"],
                                   state["q_start"], causal=case["causal"],
                                   return_lse=case["lse"])


def _turn(x, state):
    """x [tokens, heads, dim] with its leading dims turned, in float32: products and
    sums in 64 bits, for a 4-bit code may hang on the last bit."""
    case, rot = state["case"], state["case"]["rot"]
    if not rot:
        return x.float()
    cs = state["cos_sin"][state["positions"].long()].double()[:, None]
    c, s = cs[..., 0], cs[..., 1]
    part = x[..., :rot].double()
    if case["halves"]:
        a, b = part[..., :rot // 2], part[..., rot // 2:]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((turned.float(), x[..., rot:].float()), -1)


def _quantize(x, dtype):
    """Codes [..., 16 G] and scale bytes [..., G] of float32 rows [..., dim]."""
    pad = -x.shape[-1] % 32
    x = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(torch.where(torch.isfinite(top), top, torch.ones_like(top)))
    # top <= 7 * 2^e, and 7 = 0.875 * 2^3
    exponent = torch.where(mantissa <= 0.875, exponent - 3, exponent - 2)
    exponent = exponent.clamp(*EXPONENTS[dtype])
    y = torch.ldexp(x, -exponent.unsqueeze(-1))
    a = y.abs()
    code = torch.zeros(a.shape, dtype=torch.uint8, device=a.device)
    for border, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False),
                       (3.5, True), (5.0, False)):  # a tie goes up where that code is even
        code += (a >= border) if up else (a > border)
    code += (y < 0).to(torch.uint8) * 8
    code = code.flatten(-2)
    scale = torch.where(torch.isfinite(top), exponent + 127, 255).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def _values(codes, scales, dim):
    """Float32 values of rows of codes and scale bytes."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    grid = torch.cat((grid, -grid))
    pairs = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    value = grid[pairs.int()].unflatten(-1, (-1, 32))
    exponent = scales[..., :value.shape[-2]].int().sub(127).unsqueeze(-1)
    value = torch.where(exponent == 128, math.nan, torch.ldexp(value, exponent))
    return value.flatten(-2)[..., :dim]


def _read_plain(cache, case, pages=None):
    """Keys and values [pages, page_size, kv_heads, dim] of a 4-bit cache in float32."""
    kc, vc, ks, vs = (x if pages is None else x[pages] for x in _regions(cache, _groups(case)))
    return tuple(_values(c, s, case["dim"]).transpose(1, 2) for c, s in ((kc, ks), (vc, vs)))


def _run_plain(state):
    case = state["case"]
    kind, page, dtype = case["kind"], case["page"], DTYPES[case["dtype"]]
    if kind == "attend4":
        return _attend_plain(state)
    if kind == "read4":
        k, v = _read_plain(state["cache"], case, state["list"].long())
        return {"k": k.to(dtype), "v": v.to(dtype)}
    q = None if state["q"] is None else _turn(state["q"], state).to(dtype)
    k, v, slots = _turn(state["k"], state), state["v"], state["slots"]
    if kind == "rotate":
        shape = (-1, case["kv_heads"], case["dim"])
        state["k_cache"].view(shape)[slots] = k.to(dtype)
        state["v_cache"].view(shape)[slots] = v
        return {"q": q, "k_cache": state["k_cache"], "v_cache": state["v_cache"]}
    groups = _groups(case)
    kc, vc, ks, vs = _regions(state["cache"], groups)
    where, row = slots // page, slots % page
    for x, codes, scales in ((k, kc, ks), (v.float(), vc, vs)):
        c, s = _quantize(x, case["dtype"])
        codes[where, :, row] = c
        scales[where, :, row, :groups] = s
    k, v = _read_plain(state["cache"], case)
    return {"q": q, "k": k.to(dtype), "v": v.to(dtype)}


def _attend_plain(state):
    """Softmax attention in float32, padded requests side by side: as many at a time,
    and as many rows of them, as keep keys and scores under 2^30 values."""
    case, q = state["case"], state["q"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group, total = heads // kv_heads, q.shape[0]
    out = torch.zeros_like(q)
    lse = torch.full((heads, total), -math.inf, device=q.device)
    new = torch.tensor(state["new"], device=q.device)
    kv_lens, start = state["kv_lens"].long(), state["q_start"].long()
    r0, requests = 0, case["requests"]
    while r0 < requests:
        r1, longest = r0, 0
        while r1 < requests:
            m = max(longest, state["new"][r1] + state["ctx"][r1])
            if r1 > r0 and (r1 + 1 - r0) * m * kv_heads * max(dim, group) > 1 << 30:
                break
            r1, longest = r1 + 1, m
        wide = max(1, _pages(longest, page))
        rows = max(state["new"][r0:r1])
        table = state["table"][r0:r1, :wide].long().clamp_min(0)
        keys, values = _read_plain(state["cache"], case, table.flatten())
        batch, m = r1 - r0, wide * page
        keys = keys.reshape(batch, m, kv_heads, dim).permute(0, 2, 3, 1).contiguous()
        values = values.reshape(batch, m, kv_heads, dim).permute(0, 2, 1, 3).contiguous()
        # (rows of padding hold garbage: not a number times a weight of 0 stays out)
        column = torch.arange(m, device=q.device)
        held = column < kv_lens[r0:r1, None]
        values = torch.where(held[:, None, :, None], values, 0)
        step = max(1, (1 << 30) // (batch * heads * m))
        for t0 in range(0, rows, step):
            t = torch.arange(t0, min(rows, t0 + step), device=q.device)
            n = new[r0:r1, None]
            at = (start[r0:r1, None] + t).clamp_max(total - 1)
            x = q[at].float().view(batch, -1, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
            s = torch.matmul(x.reshape(batch, kv_heads, -1, dim), keys).mul_(dim ** -0.5)
            s = s.view(batch, kv_heads, group, -1, m)
            seen = held[:, None, :].expand(-1, t.numel(), -1)
            if case["causal"]:
                seen = seen & (column <= (t + kv_lens[r0:r1, None] - n)[..., None])
            s = s.masked_fill_(~seen[:, None, None], -math.inf)
            top = s.amax(-1, keepdim=True)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            s = s.sub_(top).exp_()
            weight = s.sum(-1)
            o = torch.matmul(s.view(batch, kv_heads, -1, m), values)
            o = o.view(batch, kv_heads, group, -1, dim)
            o = torch.where(weight[..., None] > 0, o / weight[..., None], torch.zeros_like(o))
            o = o.permute(0, 3, 1, 2, 4).reshape(batch, t.numel(), heads, dim)
            l = (top[..., 0] + weight.log()).reshape(batch, heads, -1)
            fresh = t < n
            out[at[fresh]] = o[fresh].to(q.dtype)
            lse[:, at[fresh]] = l.permute(1, 0, 2)[:, fresh]
        r0 = r1
    return (out, lse) if case["lse"] else out


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    new, ctx = _lengths(case)
    total, kv_heads, heads, dim = sum(new), case["kv_heads"], case["heads"], case["dim"]
    row4 = 2 * (dim / 2 + _groups(case))  # keys and values of a token and head
    if case["kind"] == "attend4":
        used = sum(n + c for n, c in zip(new, ctx) if n > 0)
        pairs = sum(n * (n + c) - (n * (n - 1) // 2 if case["causal"] else 0)
                    for n, c in zip(new, ctx))
        out = total * heads * (2 * 2 * dim + (4 if case["lse"] else 0))
        index = 4 * sum(_pages(n + c, case["page"]) for n, c in zip(new, ctx))
        return {"bytes": used * kv_heads * row4 + out + index + 8 * case["requests"],
                "flops": 4.0 * dim * heads * pairs}
    if case["kind"] == "read4":
        rows = sum(_pages(n + c, case["page"]) for n, c in zip(new, ctx)) * case["page"]
        return {"bytes": rows * kv_heads * (row4 + 4 * dim), "flops": 2.0 * rows * kv_heads * dim}
    # Queries in and out, keys and values in, a slot and a position each, the turned
    # positions' angles once.
    spots = len({p for n, c in zip(new, ctx) for p in range(c, c + n)}) if case["rot"] else 0
    size = total * (2 * 2 * heads * dim + 2 * 2 * kv_heads * dim + 8 + (4 if case["rot"] else 0))
    size += 4 * case["rot"] * spots
    flops = 3.0 * total * (heads + kv_heads) * case["rot"]
    if case["kind"] == "rotate":
        return {"bytes": size + total * 2 * 2 * kv_heads * dim, "flops": flops}
    rows = _cache_pages(case) * case["page"]
    return {"bytes": size + total * kv_heads * row4 + rows * kv_heads * (row4 + 4 * dim),
            "flops": flops + 4.0 * total * kv_heads * dim}


# ---------------------------------------------------------------------------
# The same results in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "attend4":
        return _attend_exact(state)
    if case["kind"] == "read4":
        pages = state["list"].long()
        return dict(zip("kv", (x[pages] for x in _decode(state["cache"], case))))
    q = None if state["q"] is None else _rotation(state["q"], state)
    k, v = _rotation(state["k"], state), state["v"].double()
    page, slots = case["page"], state["slots"]
    if case["kind"] == "rotate":
        names, held = ("k_cache", "v_cache"), [state["k_cache"].double(), state["v_cache"].double()]
    else:
        names, held = ("k", "v"), list(_decode(state["cache"], case))
        k, v = _nearest(k.float().double(), case), _nearest(v, case)
    out = {"q": q}
    for name, old, fresh in zip(names, held, (k, v)):
        # Row i of the cache: the token whose slot it is, or what it held.
        flat = old.reshape(-1, *old.shape[2:])
        token = torch.full((flat.shape[0],), -1, dtype=torch.int64, device="cuda")
        token.scatter_(0, slots, torch.arange(slots.numel(), device="cuda"))
        pick = fresh[token.clamp_min(0)]
        out[name] = torch.where((token >= 0)[:, None, None], pick, flat).view(old.shape)
    return out


def _rotation(x, state):
    """As complex numbers: pair (a, b) times cos + i sin."""
    case, rot = state["case"], state["case"]["rot"]
    x = x.double()
    if not rot:
        return x
    turn = torch.view_as_complex(state["cos_sin"].double())[state["positions"].long()][:, None]
    half = rot // 2
    index = torch.arange(rot, device=x.device).view(2, half).t() if case["halves"] else \
        torch.arange(rot, device=x.device).view(half, 2)
    y = torch.view_as_real(torch.view_as_complex(x[..., index].contiguous()) * turn)
    out = x.clone()
    out[..., index] = y
    return out


def _nearest(x, case):
    """The values that a 4-bit cache holds of x: multiples of the step around each."""
    dim = x.shape[-1]
    out = torch.zeros((*x.shape[:-1], 32 * _groups(case)), dtype=torch.float64, device=x.device)
    out[..., :dim] = x
    out = out.unflatten(-1, (-1, 32))
    top = out.abs().amax(-1, keepdim=True)
    low, high = EXPONENTS[case["dtype"]]
    e = torch.ceil(torch.log2(top / 7)).clamp(low, high)
    # (the logarithm may be off by one next to a power of two)
    e = torch.where(top > 7 * torch.exp2(e), e + 1, e)
    e = torch.where(top <= 7 * torch.exp2(e - 1), e - 1, e).clamp(low, high)
    y = out * torch.exp2(-e)
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0)).double()
    y = (torch.round(y / step) * step).clamp(-6, 6) * torch.exp2(e)
    return y.flatten(-2)[..., :dim]


def _decode(cache, case):
    """Keys and values [pages, page_size, kv_heads, dim] of a 4-bit cache, in 64 bits."""
    pages, heads, page, _ = cache.shape
    groups, dim = _groups(case), case["dim"]
    flat = cache.reshape(pages, heads, -1)
    d = torch.arange(dim, device=cache.device)
    row = torch.arange(page, device=cache.device)[:, None]
    for which in range(2):
        code = flat[:, :, which * page * 16 * groups + row * 16 * groups + d // 2]
        code = (code >> (4 * (d % 2)).to(torch.uint8)) & 15
        scale = flat[:, :, 2 * page * 16 * groups + which * 4 * page + row * 4 + d // 32]
        low, e = (code & 1).double(), ((code & 7) >> 1).double()
        size = torch.where(e > 0, (1 + low / 2) * torch.exp2(e - 1), low / 2)
        size = size * torch.exp2(scale.double() - 127)
        value = torch.where(code >= 8, -size, size)
        value = torch.where(scale == 255, math.nan, value)
        yield value.transpose(1, 2)


def _attend_exact(state):
    case, q = state["case"], state["q"]
    total, heads, dim = q.shape
    group, page = heads // case["kv_heads"], case["page"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full((heads, total), -math.inf, dtype=torch.float64, device=q.device)
    row = 0
    for r, (n, c) in enumerate(zip(state["new"], state["ctx"])):
        m = n + c
        pages = state["table"][r, :_pages(m, page)].long()
        k, v = (x.reshape(-1, *x.shape[2:])[:m] for x in _decode(state["cache"][pages], case))
        position = torch.arange(m, device=q.device)
        step = max(1, (1 << 27) // max(1, m))
        for h in range(case["kv_heads"]):
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            # The rows of a key head's group, token by token.
            rows = q[row:row + n, h * group:(h + 1) * group].reshape(n * group, dim)
            for i0 in range(0, n * group, step):
                i1 = min(n * group, i0 + step)
                s = (rows[i0:i1].double() * dim ** -0.5) @ kt
                token = torch.arange(i0, i1, device=q.device) // group
                head = h * group + torch.arange(i0, i1, device=q.device) % group
                if case["causal"]:
                    s = s.masked_fill(position[None] > (c + token)[:, None], -math.inf)
                total_log = torch.logsumexp(s, dim=1)
                out[row + token, head] = torch.exp(s - total_log[:, None]) @ vh
                lse[head, row + token] = total_log
        row += n
    return (out, lse) if case["lse"] else out
