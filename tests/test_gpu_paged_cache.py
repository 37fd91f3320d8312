"""The paged key/value cache on the GPU where it can go wrong: rows of one 16-byte
chunk, a free list that a captured step goes through, tokens that find no page."""

import math

import pytest
import torch

from dit_sparse_atten_amd import ops
from oracle import sequences as oracle

pytestmark = pytest.mark.gpu


def _guarded(pages, page, heads, dim, dtype, head_major, seed, device):
    """(store, cache): a cache of random rows between two guard pages of its store."""
    shape = (pages + 2, heads, page, dim) if head_major else (pages + 2, page, heads, dim)
    g = torch.Generator().manual_seed(seed)
    store = torch.randn(shape, generator=g).to(dtype).to(device)
    cache = store[1:-1]
    return store, cache.transpose(1, 2) if head_major else cache


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 8), (torch.float16, 8),
                                       (torch.float32, 4), (torch.float32, 8)], ids=str)
@pytest.mark.parametrize("heads", [1, 4, 7])
@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("first", ["valid", "none"])
def test_write_rows_of_one_chunk(cuda_device, dtype, dim, heads, head_major, first):
    """Rows of 16 bytes (one chunk a head) and of 32: every token in its own slot, the
    cache's last slot among them, nothing outside the slots."""
    page, pages, tokens = 16, 200, 2500
    g = torch.Generator().manual_seed(heads)
    slots = torch.randperm(page * pages, generator=g)[:tokens]
    last = (slots == page * pages - 1).nonzero()
    if last.numel():
        slots[last[0, 0]] = slots[0]
    slots[0] = page * pages - 1
    slots[5::11] = -1
    if first == "none":
        slots[1], slots[0] = slots[0].clone(), -1
    stores, caches = zip(*(_guarded(pages, page, heads, dim, dtype, head_major, s, cuda_device)
                           for s in (1, 2)))
    # K and V as slices of a wider projection, of wider rows.
    wide = torch.randn((tokens, 2 * heads, 2 * dim), generator=g).to(dtype).to(cuda_device)
    k, v = wide[:, :heads, :dim], wide[:, heads:, dim:]
    want = [s.clone() for s in stores]
    kept = slots >= 0
    at = slots[kept].to(cuda_device)
    for held, rows in zip(want, (k, v)):
        view = held[1:-1].transpose(1, 2) if head_major else held[1:-1]
        view[at // page, at % page] = rows[kept.to(cuda_device)]
    ops.paged_write(k, v, *caches, slots.to(cuda_device))
    for got, expected in zip(stores, want):
        assert torch.equal(got, expected)
    # Neighbours in memory, as the projection of one layer leaves them.
    for held, rows in zip(want, (k, v)):
        view = held[1:-1].transpose(1, 2) if head_major else held[1:-1]
        view[at // page, at % page] = -rows[kept.to(cuda_device)]
    ops.paged_write(-k.contiguous(), -v.contiguous(), *caches, slots.to(cuda_device))
    for got, expected in zip(stores, want):
        assert torch.equal(got, expected)


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


@pytest.mark.parametrize("start", [0, 3, 11, 12, 13, 5000, -1, -2 ** 31])
def test_plan_from_the_middle_of_the_free_list(cuda_device, start):
    """The pages behind the first `start`; none where the count leaves the list."""
    cached, new = [16, 20, 0, 5], [1, 4, 40, 100]
    table = [[7] + [-1] * 9, [3, 4] + [-1] * 8, [-1] * 10, [9] + [-1] * 9]
    free = list(range(50, 62))
    expected = oracle.plan(cached, new, table, free[start:] if 0 <= start < 12 else [], 16, 150)
    held, at = _ints(table, cuda_device), _ints([start], cuda_device)
    args = (_ints(cached, cuda_device), _ints(new, cuda_device), held, _ints(free, cuda_device),
            16, 150)
    for _ in range(2):
        got = ops.paged_plan(*args, free_start=at)
        assert [x.tolist() for x in got] == [list(x) for x in expected[:4]]
        assert held.tolist() == expected[4] and at.tolist() == [start]


def test_plan_from_refusals(cuda_device):
    def ints(*values):
        return _ints(values, cuda_device)

    table = torch.zeros((1, 2), dtype=torch.int32, device=cuda_device)
    for bad in (ints(0).long(), ints(0, 1), ints(0)[0], ints()):
        with pytest.raises(ValueError, match="free_start"):
            ops.paged_plan(ints(0), ints(1), table, ints(1, 2), 16, 1, free_start=bad)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_plan(ints(0), ints(1), table, ints(1, 2), 16, 1, free_start=ints(0).cpu())


def test_captured_step_takes_new_pages_on_every_replay(cuda_device):
    """A decoding step captured once (plan, write, attention, the free list moved on)
    and replayed 40 times: no page is held by two requests, and every output is
    attention over the whole sequence.  (Tolerance: the probabilities' rounding and
    the result's, half a step of bf16 each, of sums of at most max |v|, and half as
    much again for everything in fp32.)"""
    kh, h, dim, page, pages = 2, 8, 64, 16, 64
    lens = [15, 0, 31, 47, 30]
    requests = len(lens)
    g = torch.Generator().manual_seed(5)

    def rows(n, heads):
        return torch.randn((n, heads, dim), generator=g).to(torch.bfloat16)

    order = torch.randperm(pages, generator=g).tolist()
    k_cache = torch.full((pages, page, kh, dim), math.nan, dtype=torch.bfloat16)
    v_cache = k_cache.clone()
    keys = [rows(n, kh) for n in lens]
    values = [rows(n, kh) for n in lens]
    table = [[-1] * 8 for _ in range(requests)]
    for r, n in enumerate(lens):
        for i in range(n):
            if i % page == 0:
                table[r][i // page] = order.pop()
            k_cache[table[r][i // page], i % page] = keys[r][i]
            v_cache[table[r][i // page], i % page] = values[r][i]
    held = {"k": k_cache.to(cuda_device), "v": v_cache.to(cuda_device),
            "table": _ints(table, cuda_device), "cached": _ints(lens, cuda_device),
            "given": _ints([0], cuda_device)}
    first = {name: t.clone() for name, t in held.items()}
    free = _ints(order, cuda_device)
    new = _ints([1] * requests, cuda_device)
    q, k, v = (torch.zeros((requests, n, dim), dtype=torch.bfloat16, device=cuda_device)
               for n in (h, kh, kh))

    def step(s):
        plan = ops.paged_plan(s["cached"], new, s["table"], free, page, requests, s["given"])
        ops.paged_write(k, v, s["k"], s["v"], plan.slots)
        out, lse = ops.paged_attention(q, s["k"], s["v"], s["table"], plan.kv_lens, plan.q_start,
                                       return_lse=True)
        s["given"] += plan.status[:1]
        s["cached"].copy_(plan.kv_lens)
        return out, lse, plan.status

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step({name: t.clone() for name, t in first.items()})
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = step(held)
    for name, t in first.items():
        held[name].copy_(t)
    other = {name: t.clone() for name, t in first.items()}
    crossed = set()
    for i in range(40):
        now = [rows(requests, n) for n in (h, kh, kh)]
        for t, x in zip((q, k, v), now):
            t.copy_(x)
        graph.replay()
        out, lse, status = (t.cpu() for t in result)
        if i % 3 == 0:
            step(other)  # eager work of another cache between the replays
            torch.cuda.synchronize()
        crossed |= {r for r in range(requests) if keys[r].shape[0] % page == 0}
        assert status[1] == 0
        for r in range(requests):
            keys[r] = torch.cat((keys[r], now[1][r:r + 1]))
            values[r] = torch.cat((values[r], now[2][r:r + 1]))
        lengths = held["cached"].tolist()
        assert lengths == [x.shape[0] for x in keys]
        used = [p for row, n in zip(held["table"].tolist(), lengths)
                for p in row[:-(-n // page)]]
        assert len(set(used)) == len(used) and min(used) >= 0 and max(used) < pages, i
        expected, stat, _, _ = oracle.packed(now[0], torch.cat(keys), torch.cat(values),
                                             [1] * requests, lengths)
        v_max = max(x.abs().max().item() for x in values)
        assert (out.double() - expected).abs().max().item() <= 3 * 2 ** -8 * v_max, i
        assert (lse.double() - stat).abs().max().item() <= 2 ** -12, i
    assert crossed == set(range(requests))
    assert held["given"].item() == sum(-(-(n + 40) // page) - -(-n // page) for n in lens)


def _plan(cached, new, table, free, page, tokens, device):
    held = _ints(table, device)
    got = ops.paged_plan(_ints(cached, device), _ints(new, device), held, _ints(free, device),
                         page, tokens)
    return [x.tolist() for x in got] + [held.tolist()]


def test_plan_counts_tokens_of_a_held_page_that_is_none(cuda_device):
    """A step finds no page for its tokens; the next one has no place in that page
    either, and says so."""
    table, page = [[7, -1, -1]], 16
    *first, table = _plan([16], [4], table, [], page, 4, cuda_device)
    assert first == [[0, 4], [20], [-1] * 4, [1, 4]] and table == [[7, -1, -1]]
    # Continued all the same, with pages free again: the shared page is none.
    got = _plan([20], [1], table, [3, 5], page, 1, cuda_device)
    assert got == [[0, 1], [21], [-1], [0, 1], [[7, -1, -1]]]
    got = _plan([20], [14], table, [3, 5], page, 14, cuda_device)
    assert got == [[0, 14], [34], [-1] * 12 + [48, 49], [1, 12], [[7, -1, 3]]]
    # Made again from the same lengths, the step has its page.
    got = _plan([16], [4], table, [3, 5], page, 4, cuda_device)
    assert got == [[0, 4], [20], [48, 49, 50, 51], [1, 0], [[7, 3, -1]]]


@pytest.mark.parametrize("case", range(48))
def test_plan_with_entries_that_are_no_page(cuda_device, case):
    """Negative entries in held pages and in the free list, short lists, short rows and
    short slot maps: the plan and its counts as the oracle has them."""
    g = torch.Generator().manual_seed(1000 + case)

    def rand(lo, hi):
        return int(torch.randint(lo, hi + 1, (), generator=g))

    page = (16, 32, 128)[case % 3]
    requests = (1, 5, 64, 700)[case % 4]
    cached = [rand(0, 6 * page) for _ in range(requests)]
    new = [rand(0, (1, 3 * page)[case % 2]) for _ in range(requests)]
    need = [-(-(c + n) // page) for c, n in zip(cached, new)]
    width = max(1, max(need) - (0, 0, 2)[case % 3])
    free = [rand(0, 999) if rand(0, 3) else -rand(1, 2 ** 31 - 1) for _ in range(sum(need) + 3)]
    if case % 5 == 4:
        free = free[:len(free) // 4]
    table = [[rand(0, 10 ** 6) if rand(0, 2) else -1 for _ in range(width)]
             for _ in range(requests)]
    total = sum(new)
    tokens = (total, total + 9, total * 2 // 3)[case % 7 % 3]
    got = _plan(cached, new, table, free, page, tokens, cuda_device)
    expected = oracle.plan(cached, new, table, free, page, tokens)
    for name, a, b in zip(("q_start", "kv_lens", "slots", "status", "table"), got, expected):
        assert a == b, name


def test_plan_counts_past_31_bits(cuda_device):
    """Sums of new tokens past 2^31 are cut there, the lost ones among them."""
    most = 2 ** 31 - 1
    got = _plan([0, 0, 0], [most, most, 5], [[-1], [-1], [-1]], [5], 16, 10, cuda_device)
    assert got == [[0, most, most, most], [most, most, 5], list(range(80, 90)), [3, most],
                   [[5], [-1], [-1]]]


def test_step_that_lost_tokens_is_made_again(cuda_device):
    """Steps that advance on the device only where every token has its place: the one
    that runs out of pages leaves lengths and list as they were until a page returns."""
    page = 16
    table = _ints([[7, -1, -1], [8, -1, -1]], cuda_device)
    cached, given = _ints([16, 30], cuda_device), _ints([1], cuda_device)
    table[1, 1] = 9
    free = _ints([3, 4, 5], cuda_device)  # (3 is in use elsewhere)
    new = _ints([1, 3], cuda_device)

    def step():
        plan = ops.paged_plan(cached, new, table, free, page, 4, free_start=given)
        whole = plan.status[1:] == 0
        given.add_(plan.status[:1] * whole)
        cached.copy_(torch.where(whole, plan.kv_lens, cached))
        return plan.slots.tolist(), plan.status.tolist()

    assert step() == ([4 * 16, 9 * 16 + 14, 9 * 16 + 15, 5 * 16], [2, 0])
    assert cached.tolist() == [17, 33] and given.tolist() == [3]
    cached[0] = 32
    for _ in range(2):
        assert step() == ([-1, 5 * 16 + 1, 5 * 16 + 2, 5 * 16 + 3], [1, 1])
        assert cached.tolist() == [32, 33] and given.tolist() == [3]
    given -= 1
    free[2] = 3  # the page used elsewhere came back
    assert step() == ([3 * 16, 5 * 16 + 1, 5 * 16 + 2, 5 * 16 + 3], [1, 0])
    assert cached.tolist() == [33, 36] and given.tolist() == [3]
    assert table.tolist() == [[7, 4, 3], [8, 9, 5]]
