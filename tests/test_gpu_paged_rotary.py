"""Writes into a paged cache that turn keys and queries, 16-bit and 4-bit caches, and
the read of a 4-bit cache, against float64 oracles."""

import math

import pytest
import torch

from dit_sparse_atten_amd import ops
from oracle import fp4 as oracle

pytestmark = pytest.mark.gpu


def _angles(positions, rot, seed=0):
    angle = torch.randn((positions, rot // 2), generator=torch.Generator().manual_seed(seed),
                        dtype=torch.float64) * 10
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _inputs(tokens, heads, kv_heads, dim, dtype, seed, device):
    """Queries, keys and values as views of one projection's rows, with room behind."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, heads + 2 * kv_heads + 1, dim), generator=g).to(dtype).to(device)
    return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:-1]


def _slots(tokens, total, seed):
    """Distinct slots, the last one and places outside the cache among them."""
    slots = torch.randperm(total - 1, generator=torch.Generator().manual_seed(seed))[:tokens]
    if tokens > 2:
        slots[1] = total - 1
        slots[2::7] = torch.tensor([-1, total, -(1 << 40), 1 << 40])[
            torch.arange(len(slots[2::7])) % 4]
    return slots


def _close_turned(got, x, want, dtype):
    """One rounding to `dtype` of a sum of two products in float32: half a step of the
    value, and of each product (magnitudes up to the pair's) and their sum 2^-24."""
    pair = x.double().abs().cpu().amax(-1, keepdim=True)
    floor = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    bound = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -22 * pair + floor
    assert ((got.double().cpu() - want).abs() <= bound).all()


CASES = [(64, 8, 2, 128, 128), (1, 4, 4, 128, 64), (33, 5, 1, 80, 80), (257, 3, 3, 40, 32),
         (130, 12, 12, 96, 96), (70, 1, 1, 8, 0), (19, 2, 1, 24, 16), (300, 16, 8, 64, 16),
         (5, 7, 7, 72, 64), (1100, 9, 3, 128, 112)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", CASES)
def test_write_rotary(cuda_device, dtype, halves, tokens, heads, kv_heads, dim, rot):
    page, pages = 16, tokens // 16 + 3
    q, k, v = _inputs(tokens, heads, kv_heads, dim, dtype, tokens, cuda_device)
    cos_sin = _angles(50, rot)
    positions = torch.randint(0, 50, (tokens,), generator=torch.Generator().manual_seed(1))
    positions[3::9] = torch.tensor([-1, 50, 1 << 30, -(1 << 31)])[
        torch.arange(len(positions[3::9])) % 4]
    slots = _slots(tokens, page * pages, 2)
    # Caches between guard pages.
    stores = [torch.randn((pages + 2, page, kv_heads, dim)).to(dtype).to(cuda_device)
              for _ in range(2)]
    before = [s.clone() for s in stores]
    args = (k, v, stores[0][1:-1], stores[1][1:-1], slots.to(cuda_device),
            positions.int().to(cuda_device), cos_sin.to(cuda_device))
    turned = ops.paged_write_rotary(*args, q=q, halves=halves)
    want_q, want_k = (oracle.rotate(x, positions, cos_sin, halves) for x in (q, k))
    _close_turned(turned, q, want_q, dtype)
    bad = (positions < 0) | (positions >= 50) if rot else torch.zeros(tokens, dtype=torch.bool)
    assert torch.equal(turned[bad.to(cuda_device)], q[bad.to(cuda_device)])
    skip = (slots < 0) | (slots >= page * pages) | bad
    rows = (1 + slots // page)[~skip], (slots % page)[~skip]
    got_k, got_v = stores[0].cpu(), stores[1].cpu()
    _close_turned(got_k[rows], k[~skip.to(cuda_device)], want_k[~skip], dtype)
    assert torch.equal(got_v[rows], v.cpu()[~skip])
    for got, old in zip((got_k, got_v), before):
        old = old.cpu()
        old[rows] = got[rows]
        assert torch.equal(got, old)
    # In place, and without queries: the same bits.
    again = [b.clone() for b in before]
    own = q.clone()
    rest = (slots.to(cuda_device), positions.int().to(cuda_device), cos_sin.to(cuda_device))
    assert ops.paged_write_rotary(k, v, again[0][1:-1], again[1][1:-1], *rest, q=own, q_out=own,
                                  halves=halves) is own
    assert torch.equal(own, turned) and torch.equal(again[0], stores[0])
    again = [b.clone() for b in before]
    assert ops.paged_write_rotary(k, v, again[0][1:-1], again[1][1:-1], *rest,
                                  halves=halves) is None
    assert torch.equal(again[0], stores[0]) and torch.equal(again[1], stores[1])


def test_write_rotary_layouts(cuda_device):
    """Head-major caches and queries, slices of wider rows, rows that have to be copied,
    an output inside a larger tensor."""
    dtype, tokens, dim = torch.float16, 40, 64
    q, k, v = _inputs(tokens, 6, 2, dim, dtype, 3, cuda_device)
    cos_sin = _angles(40, dim).to(cuda_device)
    positions = torch.arange(40, dtype=torch.int32, device=cuda_device)
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(0)).to(cuda_device)[:tokens]
    plain = [torch.zeros((4, 16, 2, dim), dtype=dtype, device=cuda_device) for _ in range(2)]
    want = ops.paged_write_rotary(k, v, *plain, slots, positions, cos_sin, q=q, halves=True)
    major = [torch.zeros((4, 2, 16, dim), dtype=dtype, device=cuda_device) for _ in range(2)]
    odd = torch.zeros(tokens * 2 * dim + 1, dtype=dtype, device=cuda_device)
    odd_k = odd[1:].view(tokens, 2, dim)
    odd_k.copy_(k)
    hosted = torch.full((tokens, 9, dim + 8), 7.0, dtype=dtype, device=cuda_device)
    out = hosted[:, 2:8, :dim]
    wide = torch.zeros((40, dim // 2, 4), device=cuda_device)
    wide[..., 1:3] = cos_sin
    got = ops.paged_write_rotary(odd_k, v.transpose(0, 1).contiguous().transpose(0, 1),
                                 *[c.transpose(1, 2) for c in major], slots[torch.arange(tokens)],
                                 positions, wide[..., 1:3], q=q.transpose(0, 1).contiguous().transpose(0, 1),
                                 q_out=out, halves=True)
    assert got is out and torch.equal(out, want)
    for a, b in zip(plain, major):
        assert torch.equal(a, b.transpose(1, 2))
    out.fill_(7.0)
    assert (hosted == 7).all()


def _check_fp4(cache, before, k, v, slots, skip, dtype, dim):
    """The whole cache is what it held, with the tokens' rows in place."""
    page = cache.shape[2]
    want = [x.clone() for x in oracle.decode(before, dim)]
    rows = (slots // page)[~skip], (slots % page)[~skip]
    for held, x in zip(want, (k, v)):
        held[rows] = oracle.nearest(x, dtype)[~skip]
    for got, expected in zip(oracle.decode(cache, dim), want):
        torch.testing.assert_close(got, expected, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rot", CASES)
def test_write_fp4(cuda_device, dtype, halves, tokens, heads, kv_heads, dim, rot):
    """Codes and scales are the definition's to the bit, the rest of the cache stays."""
    page, pages = 32, tokens // 32 + 2
    q, k, v = _inputs(tokens, heads, kv_heads, dim, dtype, tokens + 1, cuda_device)
    # Magnitudes of every size, and ties: few bits.
    g = torch.Generator().manual_seed(5)
    spread = torch.exp2(torch.randint(-9, 9, (tokens, 1, 1), generator=g).float())
    k = (k * spread.to(dtype).to(cuda_device))
    v = (v * 4).round() / 4
    cos_sin = _angles(30, rot)
    positions = torch.randint(-1, 31, (tokens,), generator=g)
    slots = _slots(tokens, page * pages, 3)
    store = torch.randint(0, 250, (pages + 2, kv_heads, page, 32 * -(-dim // 32) + 8),
                          dtype=torch.uint8, generator=g).to(cuda_device)
    before, cache = store.clone(), store[1:-1]
    turn = dict(positions=positions.int().to(cuda_device), cos_sin=cos_sin.to(cuda_device))
    turned = ops.paged_write_fp4(k, v, cache, slots.to(cuda_device), q=q, halves=halves, **turn)
    bad = (positions < 0) | (positions >= 30) if rot else torch.zeros(tokens, dtype=torch.bool)
    skip = (slots < 0) | (slots >= page * pages) | bad
    want_k = oracle.rotate(k, positions, cos_sin, halves).float()
    _check_fp4(cache, before[1:-1], want_k, v, slots, skip, dtype, dim)
    assert torch.equal(store[0], before[0]) and torch.equal(store[-1], before[-1])
    _close_turned(turned, q, oracle.rotate(q, positions, cos_sin, halves), dtype)
    # Without angles: nothing turns, every token has its place.
    store.copy_(before)
    passed = ops.paged_write_fp4(k, v, cache, slots.to(cuda_device), q=q)
    assert torch.equal(passed, q)
    skip = (slots < 0) | (slots >= page * pages)
    _check_fp4(cache, before[1:-1], k.float(), v, slots, skip, dtype, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_fp4_extremes(cuda_device, dtype):
    """Zeros, the smallest and largest numbers, infinities and NaN, ties and borders of
    the exponent: what the definition says, and exactly what is read back."""
    info = torch.finfo(dtype)
    rows = [torch.zeros(64)]
    for top in (info.max, info.max * 0.87, info.smallest_normal, info.smallest_normal * info.eps,
                7.0, 7.0 * (1 + info.eps), 6.0, 6.5, 14.0, 3.5, 1e-30, 448.0,
                2.0 ** -126, 2.0 ** -127, 1.5 * 2.0 ** -125):
        x = torch.linspace(-1, 1, 64) * top
        x[40] = top
        rows.append(x)
    ties = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7] * 2)
    rows.append(torch.cat((ties, -ties)))
    rows.append(torch.cat((ties, ties / 4)))
    for value in (math.inf, -math.inf, math.nan):
        x = torch.linspace(-2, 2, 64)
        x[5] = value
        rows.append(x)
    x = torch.stack(rows).to(dtype)[:, None].to(cuda_device)
    tokens = x.shape[0]
    cache = ops.paged_cache_fp4(3, 16, 1, 64, cuda_device)
    slots = torch.arange(tokens, device=cuda_device)
    ops.paged_write_fp4(x, -x, cache, slots)
    k, v = ops.paged_read_fp4(cache, 64, dtype=dtype)
    want = oracle.nearest(x.float(), dtype)
    for got, expected in ((k, want), (v, -want)):
        got = got.reshape(-1, 1, 64)
        torch.testing.assert_close(got[:tokens].double().cpu(), expected, rtol=0, atol=0,
                                   equal_nan=True)
        assert (got[tokens:] == 0).all()


@pytest.mark.parametrize("dim", [8, 40, 64, 72, 96, 128])
@pytest.mark.parametrize("page", [16, 64, 512])
def test_read_fp4(cuda_device, dim, page):
    """Every byte pattern of codes and most of scales, listed pages in any order, twice,
    outside the cache; pages and heads of a larger cache."""
    g = torch.Generator().manual_seed(dim + page)
    row = 32 * -(-dim // 32) + 8
    whole = torch.randint(0, 256, (2, 9, 5, page, row), dtype=torch.uint8, generator=g)
    cache = whole.to(cuda_device)[1, 1:8, 1:4]
    assert not cache.is_contiguous()
    want = oracle.decode(cache, dim)
    listed = torch.tensor([3, 0, 7, 6, 3, -1, 1, 1 << 30], dtype=torch.int32)
    for dtype in (torch.bfloat16, torch.float16):
        for pages in (None, listed, listed[:0]):
            got = ops.paged_read_fp4(cache, dim, None if pages is None else pages.to(cuda_device),
                                     dtype)
            for x, values in zip(got, want):
                if pages is not None:
                    ok = (pages >= 0) & (pages < 7)
                    values = torch.where(ok[:, None, None, None],
                                         values[torch.where(ok, pages, 0).long()], 0.0)
                # (exact: the type has every element, but for fp16's range)
                assert torch.equal(torch.isnan(x.cpu()), torch.isnan(values))
                finite = ~torch.isnan(values)
                assert torch.equal(x.cpu()[finite], values[finite].to(dtype))


def test_refusals(cuda_device):
    def rows(n, h, d=64, t=torch.bfloat16):
        return torch.zeros((n, h, d), dtype=t, device=cuda_device)

    q, k = rows(4, 4), rows(4, 2)
    slots = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    turns = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    angles = _angles(5, 32).to(cuda_device)
    held = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    cache = ops.paged_cache_fp4(3, 16, 2, 64, cuda_device)

    def rotary(match, k=k, v=k, k_cache=held, v_cache=held, slots=slots, positions=turns,
               cos_sin=angles, **more):
        with pytest.raises(ValueError, match=match):
            ops.paged_write_rotary(k, v, k_cache, v_cache, slots, positions, cos_sin, **more)

    def fp4(match, k=k, v=k, cache=cache, slots=slots, positions=turns, cos_sin=angles, **more):
        with pytest.raises(ValueError, match=match):
            ops.paged_write_fp4(k, v, cache, slots, positions, cos_sin, **more)

    for refuse in (rotary, fp4):
        refuse("float32", k=rows(4, 2, t=torch.float32), v=rows(4, 2, t=torch.float32))
        refuse("like q", v=k.half())
        refuse("same shape", v=rows(4, 1))
        refuse("rows, heads", k=k[0], v=k[0])
        refuse("head", k=rows(4, 2, 136), v=rows(4, 2, 136))
        refuse("slots", slots=slots.int())
        refuse("slots", slots=slots[:3])
        refuse("CUDA", slots=slots.cpu())
        refuse("CUDA", k=k.cpu())
        refuse("positions", positions=turns.long())
        refuse("positions", positions=turns[:3])
        refuse("cos_sin", cos_sin=angles.double())
        refuse("cos_sin", cos_sin=angles[..., 0])
        refuse("CUDA", cos_sin=angles.cpu())
        refuse("turned dims", cos_sin=angles[:, :12])
        refuse("turned dims", cos_sin=_angles(5, 80).to(cuda_device))
        refuse("q must", q=rows(3, 4))
        refuse("like q", q=q.half())
        refuse("q_out needs q", q_out=q)
        refuse("q_out", q=q, q_out=k)
        refuse("expanded", q=q, q_out=q[:1].expand(4, -1, -1))
        refuse("aligned", q=q, q_out=rows(4, 4, 66)[..., :64])
        refuse("CUDA", q=q, q_out=q.cpu())
    rotary("needed", positions=None, cos_sin=None)
    rotary("k_cache", k_cache=held.half())
    rotary("heads", k_cache=held[:, :, :1], v_cache=held[:, :, :1])
    rotary("share", v_cache=held[:2])
    rotary("expanded", k_cache=held[:1].expand(3, -1, -1, -1))
    rotary("page_size", k_cache=held[:, :8], v_cache=held[:, :8])
    fp4("positions need", cos_sin=None)
    fp4("uint8", cache=held)
    fp4("uint8", cache=cache[..., :71])
    fp4("heads", cache=cache[:, :1])
    fp4("page_size", cache=cache[:, :, ::2])
    fp4("contiguous", cache=ops.paged_cache_fp4(3, 32, 2, 64, cuda_device)[:, :, ::2])
    fp4("expanded", cache=cache[:1].expand(3, -1, -1, -1))
    store = torch.zeros(3 * 2 * 16 * 72 + 8, dtype=torch.uint8, device=cuda_device)
    fp4("aligned", cache=store[8:].view(3, 2, 16, 72))
    wide = torch.zeros((3, 2 * 16 * 72 + 8), dtype=torch.uint8, device=cuda_device)
    fp4("16 bytes apart", cache=wide[:, :-8].view(3, 2, 16, 72))
    with pytest.raises(ValueError, match="float32"):
        ops.paged_read_fp4(cache, 64, dtype=torch.float32)
    with pytest.raises(ValueError, match="uint8"):
        ops.paged_read_fp4(cache, 128)
    with pytest.raises(ValueError, match="pages"):
        ops.paged_read_fp4(cache, 64, slots)
    starts, table = torch.tensor([0, 4], dtype=torch.int32, device=cuda_device), turns[:2][None]

    def attend(match, q=q, cache=cache, table=table, lens=starts[1:], starts=starts, **more):
        with pytest.raises(ValueError, match=match):
            ops.paged_attention_fp4(q, cache, table, lens, starts, **more)

    attend("uint8", cache=held)
    attend("uint8", q=rows(4, 4, 128))
    attend("share", q=rows(4, 5))
    attend("float32", q=q.float())
    attend("block_table", table=table.long())
    attend("block_table", table=table.expand(2, -1))
    attend("kv_lens", lens=starts[1:].long())
    attend("q_start", starts=starts[:1])
    attend("scale", scale=0.0)
    attend("out", out=torch.zeros_like(k))
    attend("expanded", out=q[:1].expand(4, -1, -1))
    attend("CUDA", cache=cache.cpu())
    # Nothing was written.
    torch.cuda.synchronize()
    assert (held == 0).all() and (cache == 0).all() and (q == 0).all()


def test_nothing_to_write(cuda_device):
    """No tokens, no pages, no head of queries: nothing happens but the queries' turn."""
    k = torch.ones((4, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    slots = torch.arange(4, device=cuda_device)
    turns, angles = slots.int(), _angles(5, 32).to(cuda_device)
    held = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    cache = ops.paged_cache_fp4(3, 16, 2, 64, cuda_device)
    none = ops.paged_write_rotary(k[:0], k[:0], held, held.clone(), slots[:0], turns[:0], angles,
                                  q=k[:0])
    assert none.shape == (0, 2, 64)
    ops.paged_write_fp4(k[:0], k[:0], cache, slots[:0])
    turned = ops.paged_write_rotary(k, k, held[:0], held[:0], slots, turns, angles, q=k)
    assert torch.equal(turned, ops.paged_write_fp4(k, k, cache[:0], slots, turns, angles, q=k))
    assert ops.paged_write_fp4(k, k, cache[:0], slots, turns, angles, q=k[:, :0]).shape == (4, 0, 64)
    assert (held == 0).all() and (cache == 0).all()
    got = ops.paged_read_fp4(cache[:0], 64)
    assert got[0].shape == got[1].shape == (0, 16, 2, 64)
    # One page and one head, whatever their strides.
    one = torch.as_strided(cache, (1, 1, 16, 72), (8, 24, 72, 1))
    ops.paged_write_fp4(k[:, :1], k[:, :1], one, slots)
    assert (ops.paged_read_fp4(one, 64)[0][0, :4] == 1).all()
