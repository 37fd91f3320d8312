"""Attention over a paged cache of 4-bit elements on the GPU, against the float64
oracle of the values that the cache stands for.

Tolerances as for the 16-bit cache, element by element: the probabilities are rounded to
the input type (half a step, eps / 2, relative) before they meet V, and the result once
more, |error| <= eps / 2 (sum_j p_j |v_j| + |o|); in fp16 a probability below 2^-14 of the
row's reference is off by at most 2^-25 of it.  Sums of m fp32 terms are off by m 2^-24
(of the p, and in O), 2^-18 covers the exponentials, the scaling and the joins.

Scores.  The scaled matrix instruction sums the products of 8 neighbouring dims over the
largest of them and cuts what lies 13 bits below its leading one: each of the other seven
loses less than 2^-13 of the largest product, so a score less than 7 * 2^-13 of its sum
of magnitudes S, for each of the query's terms, which are 2^-4 apart: 7 * 2^-13 * 1.07 S
with the fp32 sums' D 2^-24 S beside it (``CUT``).  Elements 2^13 below their row's
largest lose 2^-21 of that, D 2^-21 of S at most.  Where the queries are small integers
and the keys' exponents near each other nothing is cut, and the first part is 0."""

import math

import pytest
import torch

from dit_sparse_atten_amd import ops
from oracle import fp4 as oracle_fp4
from oracle import sequences as oracle

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CUT = 7 * 2.0 ** -13 * 1.07


def _check(got, lse, expected, dim, keys, v_max, cut=CUT):
    out, stat, weight, reach = expected
    step = torch.finfo(got.dtype).eps / 2
    score = ((cut + dim * 2.0 ** -21 if cut else 0.0) + dim * 2.0 ** -24) * reach
    fp32 = (torch.expm1(2 * score).t() + 2.0 * keys * 2.0 ** -24 + 2.0 ** -18)[..., None]
    bound = (step + fp32) * weight * (1 + step) + step * out.abs() + 1e-30
    if got.dtype == torch.float16:
        bound = bound + keys * 2.0 ** -25 * v_max + 2.0 ** -25
    error = (got.double().cpu() - out).abs()
    assert torch.isfinite(error).all()
    worst = (error / bound).max().item() if error.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.3f} times its bound"
    if lse is not None:
        empty = torch.isinf(stat)
        lse = lse.double().cpu()
        assert (lse[empty] == -math.inf).all()
        finite = (lse - stat)[~empty].abs()
        limit = (score + keys * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -22 * stat.abs())[~empty]
        assert (finite <= limit).all(), f"LSE off by {(finite / limit).max().item():.3f} bounds"


def _starts(lens, device):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=device)


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _rows(shape, dtype, seed, device, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype).to(device)


def _integers(shape, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-3, 4, shape, generator=g).to(dtype).to(device)


class _Cache:
    """A cache of requests in shuffled pages.  Rows past a request's length, and pages of
    none, hold bytes of every kind, scales of NaN among them."""

    def __init__(self, kv_lens, page, kv_heads, dim, seed, device, scales=(122, 128),
                 width_more=1):
        g = torch.Generator().manual_seed(seed)
        need = [-(-m // page) for m in kv_lens]
        pages, groups = sum(need) + 3, -(-dim // 32)
        order = torch.randperm(pages, generator=g).tolist()
        width = max(need + [0]) + width_more
        data = torch.randint(0, 256, (pages, kv_heads, page * (32 * groups + 8)),
                             dtype=torch.uint8, generator=g)
        data[:, :, 2 * page * 16 * groups:][torch.rand(
            (pages, kv_heads, 8 * page), generator=g) < 0.3] = 255
        self.table, at = [], 0
        code = page * 16 * groups
        for m, n in zip(kv_lens, need):
            own = order[at:at + n]
            at += n
            for i, p in enumerate(own):
                rows = min(page, m - i * page)
                for which in range(2):
                    from_byte = 2 * code + which * 4 * page
                    data[p, :, from_byte:from_byte + 4 * rows] = torch.randint(
                        *scales, (kv_heads, 4 * rows), dtype=torch.uint8, generator=g)
            self.table.append(own + [-1] * (width - n))
        # (dims past head_dim are zeros in a cache that the framework wrote)
        if dim % 32:
            codes = data[:, :, :2 * code].view(pages, kv_heads, 2 * page, groups, 16)
            codes[..., groups - 1, dim % 32 // 2:] = 0
        self.data = data.view(pages, kv_heads, page, 32 * groups + 8).to(device)
        self.dim, self.kv_lens = dim, kv_lens
        self.k, self.v = (x for x in oracle_fp4.decode(self.data, dim))

    def args(self, device):
        return (self.data, _ints(self.table, device), _ints(self.kv_lens, device))

    def expected(self, q, q_lens, causal=True, scale=None):
        return oracle.paged(q, self.k, self.v, self.table, self.kv_lens, q_lens, causal, scale)

    def v_max(self):
        return self.v.nan_to_num(0, 0, 0).abs().max().item()


HEADS = [(8, 2, 128), (4, 4, 64), (8, 1, 96), (10, 5, 40), (16, 1, 128), (3, 3, 8), (40, 40, 128)]
LENS = [
    ([1, 1, 1, 1, 1], [1, 15, 16, 17, 700]),   # a decoding step
    ([1, 0, 1], [0, 300, 5000]),               # an empty cache, no new token, a long one
    ([4, 1, 3], [4, 33, 260]),                 # a few new tokens each
    ([130, 64, 1], [130, 1000, 3]),            # chunks and a decoding request
    ([2, 50], [1, 20]),                        # more new rows than cached keys
    ([33, 127], [64, 65]),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("q_lens,kv_lens", LENS, ids=str)
def test_paged_fp4(cuda_device, dtype, page, heads, q_lens, kv_lens):
    h, kh, dim = heads
    cache = _Cache(kv_lens, page, kh, dim, 7, cuda_device)
    q = _rows((sum(q_lens), h, dim), DTYPES[dtype], 8, cuda_device)
    for causal in (True, False):
        out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device),
                                           _starts(q_lens, cuda_device), causal=causal,
                                           return_lse=True)
        _check(out, lse, cache.expected(q, q_lens, causal), dim, max(kv_lens), cache.v_max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 2], [3, 1500, 600]), ([90, 200], [90, 777])],
                         ids=str)
def test_exact_scores(cuda_device, dtype, heads, q_lens, kv_lens):
    """Small integers against keys of neighbouring exponents: no product is cut."""
    h, kh, dim = heads
    cache = _Cache(kv_lens, 32, kh, dim, 9, cuda_device, scales=(125, 127))
    q = _integers((sum(q_lens), h, dim), DTYPES[dtype], 10, cuda_device)
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts(q_lens, cuda_device),
                                       scale=0.02, return_lse=True)
    _check(out, lse, cache.expected(q, q_lens, scale=0.02), dim, max(kv_lens), cache.v_max(), 0.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,m", [(1, 300), (70, 200)])
def test_every_bit_of_the_queries(cuda_device, dtype, n, m):
    """Keys that pick one dim of the query, with scores that tell its value: every element
    enters with all of its bits (16 of them a row, within 2^4 of each other)."""
    t = DTYPES[dtype]
    dim = 128
    q = torch.zeros((n, 1, dim))
    g = torch.Generator().manual_seed(3)
    q[:, 0, ::8] = (1 + torch.rand((n, 16), generator=g)) * 2.0 ** torch.randint(
        0, 4, (n, 16), generator=g)
    q = q.to(t).to(cuda_device)
    k = torch.zeros((m, 1, dim))
    k[torch.arange(m), 0, torch.arange(m) % dim] = 1.0
    v = torch.zeros((m, 1, dim))
    v[torch.arange(m), 0, torch.arange(m) % dim] = 1.0
    cache = ops.paged_cache_fp4(-(-m // 16), 16, 1, dim, cuda_device)
    ops.paged_write_fp4(k.to(t).to(cuda_device), v.to(t).to(cuda_device), cache,
                        torch.arange(m, device=cuda_device))
    table = torch.arange(-(-m // 16), dtype=torch.int32, device=cuda_device)[None]
    out, lse = ops.paged_attention_fp4(q, cache, table, _ints([m], cuda_device),
                                       _ints([0, n], cuda_device), causal=False, scale=1.0,
                                       return_lse=True)
    expected = oracle.packed(q, k, v, [n], [m], causal=False, scale=1.0)
    _check(out, lse, expected, dim, m, 1.0, 0.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("requests,new,heads", [(37, 4, (64, 8, 128)), (34, 3, (16, 2, 64)),
                                                (4, 16, (8, 2, 128)), (2, 13, (10, 2, 40)),
                                                (5, 20, (16, 8, 96))], ids=str)
def test_a_few_tokens_each(cuda_device, requests, new, heads, causal, dtype):
    """Requests of up to 64 rows for each key head: several 16-row tiles of one, the last
    of them part of a tile, more rows than keys."""
    h, kh, dim = heads
    g = torch.Generator().manual_seed(requests)
    q_lens = torch.randint(0, new + 1, (requests,), generator=g).tolist()
    kv_lens = torch.randint(0, 300, (requests,), generator=g).tolist()
    kv_lens[1], q_lens[1] = 3500, new
    cache = _Cache(kv_lens, 32, kh, dim, 50, cuda_device)
    q = _rows((sum(q_lens), h, dim), DTYPES[dtype], 51, cuda_device)
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts(q_lens, cuda_device),
                                       causal=causal, return_lse=True)
    _check(out, lse, cache.expected(q, q_lens, causal), dim, 3500, cache.v_max())


@pytest.mark.parametrize("rows", [1, 2, 5, 9, 33])
@pytest.mark.parametrize("keys", [20000, 33333])
def test_long_split(cuda_device, rows, keys):
    """Few rows over many keys: many parts, of unequal requests."""
    kv_lens, q_lens = [keys, 129, keys // 3], [rows, rows, 1]
    cache = _Cache(kv_lens, 32, 2, 128, 11, cuda_device)
    q = _rows((sum(q_lens), 10, 128), torch.float16, 12, cuda_device, spread=0.7)
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts(q_lens, cuda_device),
                                       return_lse=True)
    _check(out, lse, cache.expected(q, q_lens), 128, keys, cache.v_max())


@pytest.mark.parametrize("n,m", [(1, 900), (3, 2500), (64, 64), (150, 700)])
def test_outlier_scores(cuda_device, n, m):
    """Scores of hundreds: the reference max moves late and by much."""
    cache = _Cache([m], 16, 2, 128, 13, cuda_device, scales=(125, 127))
    q = _integers((n, 4, 128), torch.bfloat16, 14, cuda_device)
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts([n], cuda_device),
                                       scale=2.0, return_lse=True)
    _check(out, lse, cache.expected(q, [n], scale=2.0), 128, m, cache.v_max(), 0.0)


@pytest.mark.parametrize("what", ["key", "value"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(2, 2, 128), (8, 2, 128), (4, 1, 40)], ids=str)
@pytest.mark.parametrize("n,m", [(150, 150), (4, 900), (3, 2500), (70, 3000), (1, 40)])
def test_groups_that_are_not_numbers(cuda_device, what, dtype, heads, n, m):
    """A later token's group leaves the rows before it as they are, and makes the others
    NaN: whole rows by a key, its own dims by a value."""
    h, kh, dim = heads
    page = 16
    cache = _Cache([m], page, kh, dim, 15, cuda_device)
    q = _rows((n, h, dim), DTYPES[dtype], 16, cuda_device)
    hit = m - n + n // 2  # seen by the rows from n // 2 on
    groups = -(-dim // 32)
    g = groups - 1
    at = 2 * page * 16 * groups + (4 * page if what == "value" else 0) + 4 * (hit % page) + g
    cache.data.view(cache.data.shape[0], kh, -1)[cache.table[0][hit // page], :, at] = 255
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts([n], cuda_device),
                                       return_lse=True)
    first = n // 2
    clean = cache.expected(q, [n])  # (decoded before the byte changed)
    _check(out[:first], lse[:, :first], tuple(
        x[:, :first] if i in (1, 3) else x[:first] for i, x in enumerate(clean)), dim, m,
        cache.v_max())
    if what == "key":
        assert out[first:].isnan().all() and lse[:, first:].isnan().all()
        return
    assert out[first:, :, 32 * g:].isnan().all()
    rest = tuple(x[:, first:] if i in (1, 3) else x[first:, :, :32 * g]
                 for i, x in enumerate(clean))
    _check(out[first:, :, :32 * g], lse[:, first:], rest, dim, m, cache.v_max())


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("kv_heads,row", [(4, 177), (1, 1)])
def test_query_rows_that_are_not_finite(cuda_device, kv_heads, row, value):
    n = 200 if kv_heads == 4 else 4
    cache = _Cache([200], 16, kv_heads, 64, 17, cuda_device)
    q = _rows((n, 4, 64), torch.float16, 18, cuda_device)
    args = (*cache.args(cuda_device), _starts([n], cuda_device))
    clean, stat = ops.paged_attention_fp4(q, *args, return_lse=True)
    q[row, 2, 7] = value
    out, lse = ops.paged_attention_fp4(q, *args, return_lse=True)
    assert out[row, 2].isnan().all() and lse[2, row].isnan()
    out[row, 2], lse[2, row] = clean[row, 2], stat[2, row]
    assert torch.equal(out, clean) and torch.equal(lse, stat)


@pytest.mark.parametrize("keys", [700, 2700])
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 90]], ids=str)
def test_bad_pages_take_no_part(cuda_device, q_lens, keys):
    """Entries outside the cache: -1, the page count, the type's limits."""
    kv_lens = [keys, 333]
    cache = _Cache(kv_lens, 16, 2, 128, 19, cuda_device)
    for r, i, bad in ((0, 3, -1), (0, 9, cache.data.shape[0]), (1, 9, 2 ** 31 - 1),
                      (1, 3, -2 ** 31), (0, 0, -5)):
        cache.table[r][i] = bad
    q = _rows((sum(q_lens), 4, 128), torch.bfloat16, 20, cuda_device)
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts(q_lens, cuda_device),
                                       return_lse=True)
    _check(out, lse, cache.expected(q, q_lens), 128, keys, cache.v_max())
    none = torch.full((2, 200), -1, dtype=torch.int32, device=cuda_device)
    out, lse = ops.paged_attention_fp4(q, cache.data, none, _ints(kv_lens, cuda_device),
                                       _starts(q_lens, cuda_device), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_rows_outside_every_sequence_and_lengths_that_leave_the_table(cuda_device):
    cache = _Cache([30, 5], 16, 2, 64, 21, cuda_device, width_more=0)
    q = _rows((40, 4, 64), torch.bfloat16, 22, cuda_device)
    data, table, lens = cache.args(cuda_device)
    starts = _ints([3, 14, 31], cuda_device)
    out, lse = ops.paged_attention_fp4(q, data, table, lens, starts, return_lse=True)
    _check(out[3:31], lse[:, 3:31], cache.expected(q[3:31], [11, 17]), 64, 30, cache.v_max())
    outside = torch.ones(40, dtype=torch.bool, device=cuda_device)
    outside[3:31] = False
    assert (out[outside] == 0).all() and (lse[:, outside] == -math.inf).all()
    given = torch.full_like(q, 7.0)
    result, again = ops.paged_attention_fp4(q, data, table, lens, starts, out=given,
                                            return_lse=True)
    assert result is given and (given[outside] == 7.0).all()
    assert torch.equal(given[3:31], out[3:31]) and torch.equal(lse, again)
    # Lengths past the table's width are cut to it, negative ones to 0.
    one = ops.paged_attention_fp4(q[:2], data, table, _ints([10 ** 9, -3], cuda_device),
                                  _ints([0, 1, 2], cuda_device))
    # (the two rows past the request's own 30 hold groups that are not numbers)
    torch.testing.assert_close(one, ops.paged_attention_fp4(
        q[:2], data, table, _ints([32, 0], cuda_device), _ints([0, 1, 2], cuda_device)),
        rtol=0, atol=0, equal_nan=True)
    assert (one[1] == 0).all()
    # No request, no page, no row.
    none = ops.paged_attention_fp4(q[:3], data, table[:0], lens[:0], _ints([0], cuda_device))
    assert (none == 0).all()
    none = ops.paged_attention_fp4(q[:2], data[:0], table, lens, _ints([0, 1, 2], cuda_device))
    assert (none == 0).all()
    assert ops.paged_attention_fp4(q[:0], data, table, lens,
                                   _ints([0, 0, 0], cuda_device)).shape == (0, 4, 64)


def test_layouts(cuda_device):
    """Pages and heads of a larger cache, queries and outputs of other strides, copied
    where they have to be, an output over q."""
    cache = _Cache([60, 7], 16, 2, 128, 23, cuda_device)
    fused = _rows((2, 8, 128), torch.bfloat16, 24, cuda_device)
    q = fused[:, 2:6]
    rest = (_ints(cache.table, cuda_device), _ints([60, 7], cuda_device),
            _ints([0, 1, 2], cuda_device))
    base = ops.paged_attention_fp4(q.contiguous(), cache.data, *rest)
    pages = cache.data.shape[0]
    larger = torch.randint(0, 256, (3, pages, 5, 16, 136), dtype=torch.uint8, device=cuda_device)
    larger[1, :, 2:4] = cache.data
    view = larger[1, :, 2:4]
    holder = torch.zeros((2, 6, 160), dtype=torch.bfloat16, device=cuda_device)
    out = holder[:, 1:5, 16:144]
    ops.paged_attention_fp4(q, view, *rest, out=out)
    assert torch.equal(out, base) and (holder[:, 0] == 0).all() and (holder[:, :, :16] == 0).all()
    odd = torch.zeros((2, 4, 129), dtype=torch.bfloat16, device=cuda_device)
    odd[..., :128] = q
    assert torch.equal(base, ops.paged_attention_fp4(odd[..., :128], view, *rest))
    own = q.contiguous()
    assert ops.paged_attention_fp4(own, view, *rest, out=own) is own
    assert torch.equal(own, base)


def test_cache_past_32_bits(cuda_device):
    """A cache of more than 2^32 bytes: pages at its far end."""
    pages, page, kh, dim = 16500, 256, 8, 128
    small = _Cache([400, 512], page, kh, dim, 25, cuda_device)
    data = torch.zeros((pages, kh, page, 136), dtype=torch.uint8, device=cuda_device)
    assert data.numel() > 1 << 32
    own = [16499, 0, 16000, 15900]
    for far, near in zip(own, small.table[0][:2] + small.table[1][:2]):
        data[far] = small.data[near]
    table = _ints([own[:2], own[2:]], cuda_device)
    for lens in ([1, 60], [1, 1]):
        q = _rows((sum(lens), kh, dim), torch.bfloat16, 26, cuda_device)
        out, lse = ops.paged_attention_fp4(q, data, table, _ints([400, 512], cuda_device),
                                           _starts(lens, cuda_device), return_lse=True)
        _check(out, lse, small.expected(q, lens), dim, 512, small.v_max())
    new = _rows((3, kh, dim), torch.bfloat16, 27, cuda_device)
    slots = torch.tensor([pages * page - 1, -1, 16100 * page + 17], device=cuda_device)
    ops.paged_write_fp4(new, -new, data, slots)
    k, v = ops.paged_read_fp4(data, dim, _ints([pages - 1, 16100], cuda_device))
    want = oracle_fp4.nearest(new.float(), torch.bfloat16)
    assert torch.equal(k[0, -1].double().cpu(), want[0])
    assert torch.equal(v[1, 17].double().cpu(), -want[2])
    assert (k[1, 16] == 0).all() and (k[1, 18] == 0).all()


def test_repeats_bit_for_bit(cuda_device):
    kv_lens = [5000, 800, 33, 2100]
    cache = _Cache(kv_lens, 16, 2, 128, 28, cuda_device)
    q = _rows((200, 8, 128), torch.bfloat16, 29, cuda_device)
    for lens in ([1, 1, 1, 1], [30, 100, 3, 67]):
        args = (q[:sum(lens)], *cache.args(cuda_device), _starts(lens, cuda_device))
        first = ops.paged_attention_fp4(*args, return_lse=True)
        for _ in range(5):
            again = ops.paged_attention_fp4(*args, return_lse=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("requests", [65, 1025, 3000])
def test_many_requests(cuda_device, requests):
    g = torch.Generator().manual_seed(requests)
    kv_lens = torch.randint(0, 60, (requests,), generator=g).tolist()
    q_lens = [int(i % 7 != 3) for i in range(requests)]
    cache = _Cache(kv_lens, 16, 1, 64, 30, cuda_device)
    q = _rows((sum(q_lens), 4, 64), torch.bfloat16, 31, cuda_device)
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts(q_lens, cuda_device),
                                       return_lse=True)
    _check(out, lse, cache.expected(q, q_lens), 64, 60, cache.v_max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("requests,heads", [(300, (8, 1, 128)), (43, (12, 6, 40)),
                                            (33, (8, 8, 64)), (7, (64, 64, 96))], ids=str)
def test_more_tiles_than_compute_units(cuda_device, dtype, requests, heads):
    """Chains of short and long tiles, one cut over many chains, requests without keys or
    new tokens, pages outside the cache."""
    h, kh, dim = heads
    g = torch.Generator().manual_seed(requests)
    kv_lens = torch.randint(0, 400, (requests,), generator=g).tolist()
    kv_lens[2], kv_lens[5] = 6000, 1700
    q_lens = [int(i % 7 != 3) for i in range(requests)]
    cache = _Cache(kv_lens, 16, kh, dim, 32, cuda_device)
    cache.table[2][200] = cache.table[5][0] = -1
    q = _rows((sum(q_lens), h, dim), DTYPES[dtype], 33, cuda_device)
    args = (q, *cache.args(cuda_device), _starts(q_lens, cuda_device))
    out, lse = ops.paged_attention_fp4(*args, return_lse=True)
    _check(out, lse, cache.expected(q, q_lens), dim, 6000, cache.v_max())
    again = ops.paged_attention_fp4(*args, return_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_more_key_heads_than_chains(cuda_device):
    kv_lens = [1500, 0, 40]
    cache = _Cache(kv_lens, 16, 600, 8, 34, cuda_device)
    q = _rows((3, 600, 8), torch.bfloat16, 35, cuda_device)
    out, lse = ops.paged_attention_fp4(q, *cache.args(cuda_device), _starts([1] * 3, cuda_device),
                                       return_lse=True)
    _check(out, lse, cache.expected(q, [1, 1, 1]), 8, 1500, cache.v_max())


def _angles(positions, rot):
    rate = 100.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _positions(plan, cached, tokens):
    token = torch.arange(tokens, device=cached.device)
    r = torch.searchsorted(plan.q_start[1:], token, right=True).clamp_max(cached.shape[0] - 1)
    return (cached[r] + token - plan.q_start[r]).int()


@pytest.mark.parametrize("halves", [False, True])
def test_prompts_chunks_and_steps(cuda_device, halves):
    """Plan, rotated write and attention of prompts, a chunk and single tokens, in both
    kinds of cache, against whole sequences turned at once."""
    kh, h, dim, rot, page = 2, 8, 128, 96, 16
    steps = [[37, 5, 0, 210], [64, 1, 30, 3], [1, 1, 1, 1], [1, 0, 1, 1], [1, 1, 0, 1]]
    whole = [sum(s[r] for s in steps) for r in range(4)]
    g = torch.Generator().manual_seed(60)
    q, k, v = ([torch.randn((n, heads, dim), generator=g).to(torch.bfloat16).to(cuda_device)
                for n in whole] for heads in (h, kh, kh))
    angles = _angles(300, rot)
    pages = 60
    cache = ops.paged_cache_fp4(pages, page, kh, dim, cuda_device)
    k_cache = torch.full((pages, page, kh, dim), math.nan, dtype=torch.bfloat16,
                         device=cuda_device)
    v_cache = k_cache.clone()
    table = torch.full((4, 20), -1, dtype=torch.int32, device=cuda_device)
    free = torch.randperm(pages, generator=g).to(torch.int32).to(cuda_device)
    cached = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    done, parts = [0] * 4, [[[] for _ in range(4)] for _ in range(2)]
    for new in steps:
        pick = [slice(d, d + n) for d, n in zip(done, new)]
        qs, ks, vs = (torch.cat([x[r][pick[r]] for r in range(4)]) for x in (q, k, v))
        qs, ks, vs = (torch.cat((x, x[:1].expand(3, -1, -1))) for x in (qs, ks, vs))
        plan = ops.paged_plan(cached, _ints(new, cuda_device), table, free, page, sum(new) + 3)
        positions = _positions(plan, cached, sum(new) + 3)
        turn = (plan.slots, positions, angles.to(cuda_device))
        turned = ops.paged_write_rotary(ks, vs, k_cache, v_cache, *turn, q=qs, halves=halves)
        again = ops.paged_write_fp4(ks, vs, cache, *turn, q=qs, q_out=qs, halves=halves)
        assert again is qs and torch.equal(again, turned)
        seen = (table, plan.kv_lens, plan.q_start)
        outs = (ops.paged_attention(turned, k_cache, v_cache, *seen),
                ops.paged_attention_fp4(turned, cache, *seen))
        for out, own in zip(outs, parts):
            assert (out[sum(new):] == 0).all()
            for r, part in enumerate(out[:sum(new)].split(new)):
                own[r].append(part)
        taken, lost = plan.status.tolist()
        assert lost == 0
        free, cached = free[taken:], plan.kv_lens
        done = [d + n for d, n in zip(done, new)]
    at = torch.cat([torch.arange(n) for n in whole])
    allq, allk = (oracle_fp4.rotate(torch.cat(x), at, angles, halves) for x in (q, k))
    allq = allq.to(torch.bfloat16)  # (as a write hands them on: half a step, in q and keys,
    step = torch.finfo(torch.bfloat16).eps / 2  # two of them where float32 is next to a border)
    for which, own in enumerate(parts):
        got = torch.cat([torch.cat(p) for p in own])
        if which == 0:
            keys, values, cut = allk, torch.cat(v).double().cpu(), 3 * step
        else:
            keys = oracle_fp4.nearest(allk.float(), torch.bfloat16)
            values, cut = oracle_fp4.nearest(torch.cat(v).float(), torch.bfloat16), CUT + 2 * step
        expected = oracle.packed(allq, keys, values, whole)
        _check(got, None, expected, dim, max(whole), values.abs().max().item(), cut)


def test_captured_step_replays_with_new_lengths(cuda_device):
    """A decoding step captured once (plan, positions, rotated write, attention) and
    replayed as the requests grow, eager steps of another cache between the replays."""
    kh, h, dim, page, requests, pages = 2, 8, 64, 16, 5, 64
    angles = _angles(200, dim).to(cuda_device)

    def caches():
        g = torch.Generator().manual_seed(70)
        data = torch.randint(0, 256, (pages, kh, page * 72), dtype=torch.uint8, generator=g)
        data[:, :, 64 * page:] = data[:, :, 64 * page:] % 8 + 122
        return {"cache": data.view(pages, kh, page, 72).to(cuda_device),
                "table": torch.arange(requests * 8, dtype=torch.int32,
                                      device=cuda_device).view(requests, 8).clone(),
                "free": torch.arange(40, 64, dtype=torch.int32, device=cuda_device),
                "given": _ints([0], cuda_device),
                "cached": _ints([3, 0, 100, 47, 16], cuda_device)}

    new = _ints([1] * requests, cuda_device)
    q, k, v = (torch.empty((requests, n, dim), dtype=torch.bfloat16, device=cuda_device)
               for n in (h, kh, kh))

    def step(s):
        plan = ops.paged_plan(s["cached"], new, s["table"], s["free"], page, requests,
                              free_start=s["given"])
        turned = ops.paged_write_fp4(k, v, s["cache"], plan.slots,
                                     _positions(plan, s["cached"], requests), angles, q=q)
        out, lse = ops.paged_attention_fp4(turned, s["cache"], s["table"], plan.kv_lens,
                                           plan.q_start, return_lse=True)
        s["cached"].copy_(plan.kv_lens)
        s["given"] += plan.status[:1]
        return out, lse

    def inputs(i):
        for n, t in enumerate((q, k, v)):
            t.copy_(_rows(t.shape, t.dtype, 71 + 3 * i + n, cuda_device))

    eager, captured, warm = caches(), caches(), caches()
    inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(captured)
    for name, t in caches().items():  # what the capture's own pass may have left
        captured[name].copy_(t)
    for i in range(20):
        inputs(i)
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        expected = step(eager)
        assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1]), i
        for name in ("cache", "table", "cached", "given"):
            assert torch.equal(eager[name], captured[name]), (i, name)


def test_captured_step_of_many_tiles(cuda_device):
    """Chains and joins of a captured call follow the lengths of each replay."""
    requests, kh, h, dim = 40, 8, 16, 128
    cache = _Cache([2500] + [200] * (requests - 1), 16, kh, dim, 36, cuda_device)
    data, table, lens = cache.args(cuda_device)
    q = _rows((requests, h, dim), torch.bfloat16, 37, cuda_device)
    start = _starts([1] * requests, cuda_device)

    def call():
        return ops.paged_attention_fp4(q, data, table, lens, start, return_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for i in range(6):
        kv_lens = [(0, 2500, 3, 1111, 2499, 700)[i]] + [(37 * r + 91 * i) % 201
                                                        for r in range(1, requests)]
        lens.copy_(_ints(kv_lens, cuda_device))
        q.copy_(_rows(q.shape, q.dtype, 38 + i, cuda_device))
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        expected = call()
        assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1]), i
        cache.kv_lens = kv_lens
        _check(got[0], got[1], cache.expected(q, [1] * requests), dim, 2500, cache.v_max())


def test_calls_on_two_streams_and_two_graphs(cuda_device):
    """Calls that overlap, and graphs replayed in turn, keep their workspaces apart."""
    kv_lens = [9000, 500]
    cache = _Cache(kv_lens, 16, 2, 128, 32, cuda_device)
    at = cache.args(cuda_device)
    q = [_rows((n, 8, 128), torch.bfloat16, 33 + n, cuda_device) for n in (2, 90)]
    starts = [_starts([1, 1], cuda_device), _starts([60, 30], cuda_device)]
    expected = [ops.paged_attention_fp4(x, *at, s) for x, s in zip(q, starts)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(ops.paged_attention_fp4(q[i], *at, starts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, expected[i]) for r in results[i])
    graphs, outs = [], []
    for x, s in zip(q, starts):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.paged_attention_fp4(x, *at, s))
        graphs.append(graph)
    for i in range(6):
        graphs[i % 2].replay()
        ops.paged_attention_fp4(q[1], *at, starts[1])
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, expected):
            assert torch.equal(out, want), i
