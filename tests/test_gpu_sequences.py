"""Sequences of different lengths on the GPU: the page plan, the cache write,
attention over packed prompts and over a paged cache, against the float64 oracle.

Tolerances, element by element.  The probabilities are rounded to the input type
(half a step, eps / 2, relative) before they meet V, and the result once more:
|error| <= eps / 2 (sum_j p_j |v_j| + |o|).  In fp16 a probability below 2^-14 of
the row's reference is off by at most 2^-25 of it, m keys of them by m 2^-25
max|v|.  The fp32 part: a score is a sum of D products, off by at most D 2^-24
times its sum of magnitudes S, so every p by a factor e^(2 D 2^-24 S), and sums of
m fp32 terms by m 2^-24, taken once for the sum of the p and once for O; 2^-18 for
the exponentials, the scaling and the joins."""

import math

import pytest
import torch

from dit_sparse_atten_amd import ops
from oracle import sequences as oracle

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _check(got, lse, expected, dim, keys, v_max):
    out, stat, weight, reach = expected
    step = torch.finfo(got.dtype).eps / 2
    # Relative error of a row's sums in fp32, [rows, heads, 1].
    fp32 = (2.0 * dim * 2.0 ** -24 * reach.t() + 2.0 * keys * 2.0 ** -24 + 2.0 ** -18)[..., None]
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
        limit = (dim * 2.0 ** -24 * reach + keys * 2.0 ** -24 + 2.0 ** -18
                 + 2.0 ** -22 * stat.abs())[~empty]
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


def _cache(kv_lens, page, kv_heads, dim, dtype, seed, device, width_more=1, unused="nan"):
    """Caches and table of requests in shuffled pages; rows past a request's
    length, and pages of none, hold `unused` values."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-m // page) for m in kv_lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g).tolist()
    width = max(need + [0]) + width_more
    table, at = [], 0
    fill = math.nan if unused == "nan" else 0.0
    k = torch.full((pages, page, kv_heads, dim), fill, dtype=dtype)
    v = torch.full((pages, page, kv_heads, dim), fill, dtype=dtype)
    for m, n in zip(kv_lens, need):
        own = order[at:at + n]
        at += n
        for i, p in enumerate(own):
            rows = min(page, m - i * page)
            k[p, :rows] = torch.randn((rows, kv_heads, dim), generator=g).to(dtype)
            v[p, :rows] = torch.randn((rows, kv_heads, dim), generator=g).to(dtype)
        table.append(own + [-1] * (width - n))
    return k.to(device), v.to(device), table


# (heads, kv_heads, head_dim): groups of 1 to 16, dims below and between 64 and 128.
HEADS = [(4, 4, 128), (8, 2, 128), (12, 12, 64), (7, 1, 96), (10, 2, 40), (16, 1, 128), (3, 3, 8)]
LENGTHS = [
    [1], [64], [65, 0, 1], [127, 128, 129], [0, 0, 5, 0], [33, 300, 2, 17], [1, 1, 1, 2, 1],
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_packed_self(cuda_device, dtype, heads, lens):
    h, kh, dim = heads
    t = DTYPES[dtype]
    total = sum(lens)
    q = _rows((total, h, dim), t, 1, cuda_device)
    k = _rows((total, kh, dim), t, 2, cuda_device)
    v = _rows((total, kh, dim), t, 3, cuda_device)
    for causal in (True, False):
        out, lse = ops.packed_attention(q, k, v, _starts(lens, cuda_device), causal=causal,
                                        return_lse=True)
        _check(out, lse, oracle.packed(q, k, v, lens, causal=causal), dim, max(lens),
               v.abs().max().item())


@pytest.mark.parametrize("q_lens,k_lens", [
    ([5, 1, 40], [200, 64, 40]),       # rows at the end of more keys
    ([70, 3, 9], [10, 0, 1]),          # more rows than keys: the first see none
    ([1, 1, 1], [1000, 0, 257]),       # single rows
    ([0, 130, 0], [50, 131, 7]),       # sequences without rows
    ([260], [4000]),                   # split along the keys
], ids=str)
@pytest.mark.parametrize("heads", [(8, 2, 128), (5, 5, 64), (6, 1, 80)], ids=str)
def test_packed_other_key_lengths(cuda_device, q_lens, k_lens, heads):
    h, kh, dim = heads
    q = _rows((sum(q_lens), h, dim), torch.bfloat16, 4, cuda_device)
    k = _rows((sum(k_lens), kh, dim), torch.bfloat16, 5, cuda_device)
    v = _rows((sum(k_lens), kh, dim), torch.bfloat16, 6, cuda_device)
    for causal in (True, False):
        out, lse = ops.packed_attention(q, k, v, _starts(q_lens, cuda_device),
                                        _starts(k_lens, cuda_device), causal=causal,
                                        return_lse=True)
        _check(out, lse, oracle.packed(q, k, v, q_lens, k_lens, causal), dim, max(k_lens),
               v.abs().max().item())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (8, 1, 96), (10, 5, 40), (40, 40, 128)], ids=str)
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([1, 1, 1, 1, 1], [1, 15, 16, 17, 700]),   # a decoding step
    ([1, 0, 1], [0, 300, 5000]),               # an empty cache, no new token, a long one
    ([4, 1, 3], [4, 33, 260]),                 # a few new tokens each
    ([130, 64, 1], [130, 1000, 3]),            # chunks and a decoding request
    ([2, 50], [1, 20]),                        # more new rows than cached keys
], ids=str)
def test_paged(cuda_device, dtype, page, heads, q_lens, kv_lens):
    h, kh, dim = heads
    t = DTYPES[dtype]
    k_cache, v_cache, table = _cache(kv_lens, page, kh, dim, t, 7, cuda_device)
    q = _rows((sum(q_lens), h, dim), t, 8, cuda_device)
    v_max = v_cache[~v_cache.isnan()].abs().max().item() if sum(kv_lens) else 0.0
    for causal in (True, False):
        out, lse = ops.paged_attention(q, k_cache, v_cache, _ints(table, cuda_device),
                                       _ints(kv_lens, cuda_device), _starts(q_lens, cuda_device),
                                       causal=causal, return_lse=True)
        _check(out, lse, oracle.paged(q, k_cache, v_cache, table, kv_lens, q_lens, causal), dim,
               max(kv_lens), v_max)


@pytest.mark.parametrize("rows", [1, 2, 5, 9, 33])
@pytest.mark.parametrize("keys", [20000, 33333])
def test_paged_long_split(cuda_device, rows, keys):
    """Few rows over many keys: many parts, of unequal requests."""
    kv_lens, q_lens = [keys, 129, keys // 3], [rows, rows, 1]
    k_cache, v_cache, table = _cache(kv_lens, 32, 2, 128, torch.float16, 9, cuda_device)
    q = _rows((sum(q_lens), 10, 128), torch.float16, 10, cuda_device, spread=1.5)
    out, lse = ops.paged_attention(q, k_cache, v_cache, _ints(table, cuda_device),
                                   _ints(kv_lens, cuda_device), _starts(q_lens, cuda_device),
                                   return_lse=True)
    _check(out, lse, oracle.paged(q, k_cache, v_cache, table, kv_lens, q_lens), 128, keys,
           v_cache[~v_cache.isnan()].abs().max().item())


@pytest.mark.parametrize("keys", [64, 300])
def test_outlier_scores(cuda_device, keys):
    """Scores of +-400: the reference max moves late and by much, rows hold one
    probability near 1."""
    q = _rows((keys, 4, 128), torch.bfloat16, 11, cuda_device, spread=6.0)
    k = _rows((keys, 2, 128), torch.bfloat16, 12, cuda_device, spread=6.0)
    v = _rows((keys, 2, 128), torch.bfloat16, 13, cuda_device)
    out, lse = ops.packed_attention(q, k, v, _starts([keys], cuda_device), return_lse=True)
    _check(out, lse, oracle.packed(q, k, v, [keys]), 128, keys, v.abs().max().item())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("group", [1, 4])
def test_hidden_values_do_not_reach_earlier_rows(cuda_device, value, group):
    """A later token's key and value that are not finite leave earlier rows as
    they are (packed and paged, wide and narrow tiles, whole and split keys)."""
    for n, m in ((150, 150), (4, 900), (3, 2500), (70, 3000)):
        q = _rows((n, 2 * group, 128), torch.bfloat16, 14, cuda_device)
        k = _rows((m, 2, 128), torch.bfloat16, 15, cuda_device)
        v = _rows((m, 2, 128), torch.bfloat16, 16, cuda_device)
        hit = m - n + n // 2  # seen by the rows from n // 2 on
        k[hit, :, 5] = value
        v[hit, :, ::3] = value
        starts = (_starts([n], cuda_device), _starts([m], cuda_device))
        clean = oracle.packed(q, k, v, [n], [m])
        out, lse = ops.packed_attention(q, k, v, *starts, return_lse=True)
        first = n // 2
        _check(out[:first], lse[:, :first], tuple(
            x[:, :first] if i in (1, 3) else x[:first] for i, x in enumerate(clean)), 128, m, 6.0)
        pages = -(-m // 16)
        pad = torch.zeros((pages * 16 - m, 2, 128), dtype=k.dtype, device=cuda_device)
        kc = torch.cat((k, pad)).view(pages, 16, 2, 128)
        vc = torch.cat((v, pad)).view(pages, 16, 2, 128)
        table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
        paged, paged_lse = ops.paged_attention(q, kc, vc, table, _ints([m], cuda_device),
                                               starts[0], return_lse=True)
        _check(paged[:first], paged_lse[:, :first], tuple(
            x[:, :first] if i in (1, 3) else x[:first] for i, x in enumerate(clean)), 128, m, 6.0)
        # Finite scores, a value that is not: the rows that see it have it.
        k[hit, :, 5] = 0.5
        out = ops.packed_attention(q, k, v, *starts)
        assert torch.isfinite(out[:first].float()).all()
        assert not torch.isfinite(out[first:, :, ::3].float()).any()
        assert torch.isfinite(out[first:, :, 1::3].float()).all()


@pytest.mark.parametrize("kv_heads,row", [(4, 177), (1, 1)])
def test_nan_query_row_stays_alone(cuda_device, kv_heads, row):
    """(200 rows, and 4 of them as four heads of one key head: both tile heights)"""
    n = 200 if kv_heads == 4 else 4
    q = _rows((n, 4, 64), torch.float16, 17, cuda_device)
    k = _rows((200, kv_heads, 64), torch.float16, 18, cuda_device)
    v = _rows((200, kv_heads, 64), torch.float16, 19, cuda_device)
    starts = _starts([n], cuda_device), _starts([200], cuda_device)
    clean, stat = ops.packed_attention(q, k, v, *starts, return_lse=True)
    q[row, 2] = math.nan
    out, lse = ops.packed_attention(q, k, v, *starts, return_lse=True)
    assert out[row, 2].isnan().all() and lse[2, row].isnan()
    out[row, 2], lse[2, row] = clean[row, 2], stat[2, row]
    assert torch.equal(out, clean) and torch.equal(lse, stat)


def test_rows_outside_every_sequence(cuda_device):
    """A padded batch: rows before the first and behind the last sequence are 0
    in a new output and untouched in a given one."""
    q = _rows((40, 4, 64), torch.bfloat16, 20, cuda_device)
    k = _rows((40, 2, 64), torch.bfloat16, 21, cuda_device)
    v = _rows((40, 2, 64), torch.bfloat16, 22, cuda_device)
    starts = _ints([3, 3, 20, 31], cuda_device)
    expected = oracle.packed(q[3:31], k[3:31], v[3:31], [0, 17, 11])
    out, lse = ops.packed_attention(q, k, v, starts, return_lse=True)
    _check(out[3:31], lse[:, 3:31], expected, 64, 17, v.abs().max().item())
    outside = torch.ones(40, dtype=torch.bool, device=cuda_device)
    outside[3:31] = False
    assert (out[outside] == 0).all() and (lse[:, outside] == -math.inf).all()
    given = torch.full_like(q, 7.0)
    result, lse2 = ops.packed_attention(q, k, v, starts, out=given, return_lse=True)
    assert result is given and (given[outside] == 7.0).all()
    assert torch.equal(given[3:31], out[3:31]) and torch.equal(lse, lse2)
    k_cache, v_cache, table = _cache([30, 5], 16, 2, 64, torch.bfloat16, 23, cuda_device)
    out, lse = ops.paged_attention(q, k_cache, v_cache, _ints(table, cuda_device),
                                   _ints([30, 5], cuda_device), _ints([0, 1, 2], cuda_device),
                                   return_lse=True)
    assert (out[2:] == 0).all() and (lse[:, 2:] == -math.inf).all()
    assert (out[:2] != 0).any()


def test_starts_that_leave_the_tensors(cuda_device):
    """Starts and lengths past the tensors are cut to them."""
    q = _rows((50, 4, 64), torch.bfloat16, 24, cuda_device)
    k = _rows((50, 4, 64), torch.bfloat16, 25, cuda_device)
    v = _rows((50, 4, 64), torch.bfloat16, 26, cuda_device)
    out = ops.packed_attention(q, k, v, _ints([0, 20, 5000], cuda_device))
    assert torch.equal(out, ops.packed_attention(q, k, v, _ints([0, 20, 50], cuda_device)))
    out = ops.packed_attention(q, k, v, _ints([-7, 20, 50], cuda_device))
    assert torch.equal(out, ops.packed_attention(q, k, v, _ints([0, 20, 50], cuda_device)))
    k_cache, v_cache, table = _cache([32], 16, 4, 64, torch.bfloat16, 27, cuda_device,
                                     width_more=0)
    at = (_ints(table, cuda_device),)
    long = ops.paged_attention(q[:1], k_cache, v_cache, *at, _ints([10 ** 6], cuda_device),
                               _ints([0, 1], cuda_device))
    assert torch.equal(long, ops.paged_attention(q[:1], k_cache, v_cache, *at,
                                                 _ints([32], cuda_device),
                                                 _ints([0, 1], cuda_device)))
    none = ops.paged_attention(q[:1], k_cache, v_cache, *at, _ints([-3], cuda_device),
                               _ints([0, 1], cuda_device))
    assert (none == 0).all()


@pytest.mark.parametrize("keys", [700, 2700])
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 90]], ids=str)
def test_bad_pages_take_no_part(cuda_device, q_lens, keys):
    """Entries outside the cache: -1, the page count, the type's limits (the longer
    request's keys are cut into parts)."""
    kv_lens = [keys, 333]
    k_cache, v_cache, table = _cache(kv_lens, 16, 2, 128, torch.bfloat16, 28, cuda_device)
    for r, bad in ((0, -1), (0, k_cache.shape[0]), (1, 2 ** 31 - 1), (1, -2 ** 31)):
        table[r][3 if bad < 0 else 9] = bad
    table[0][0] = -5
    q = _rows((sum(q_lens), 4, 128), torch.bfloat16, 29, cuda_device)
    out, lse = ops.paged_attention(q, k_cache, v_cache, _ints(table, cuda_device),
                                   _ints(kv_lens, cuda_device), _starts(q_lens, cuda_device),
                                   return_lse=True)
    _check(out, lse, oracle.paged(q, k_cache, v_cache, table, kv_lens, q_lens), 128, keys,
           v_cache[~v_cache.isnan()].abs().max().item())
    # A table of none but bad pages: rows without a key.
    out, lse = ops.paged_attention(q, k_cache, v_cache,
                                   torch.full((2, 200), -1, dtype=torch.int32, device=cuda_device),
                                   _ints(kv_lens, cuda_device), _starts(q_lens, cuda_device),
                                   return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_no_sequences_rows_or_keys(cuda_device):
    def rows(n, h, d=64):
        return _rows((n, h, d), torch.bfloat16, 30, cuda_device)

    none = _ints([0], cuda_device)
    out, lse = ops.packed_attention(rows(0, 4), rows(0, 2), rows(0, 2), none, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    out = ops.packed_attention(rows(5, 4), rows(5, 2), rows(5, 2), none)
    assert (out == 0).all()
    out = ops.packed_attention(rows(5, 4), rows(0, 2), rows(0, 2), _ints([0, 5], cuda_device),
                               _ints([0, 0], cuda_device))
    assert (out == 0).all()
    empty = torch.empty((0, 16, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    out = ops.paged_attention(rows(2, 4), empty, empty,
                              torch.zeros((2, 3), dtype=torch.int32, device=cuda_device),
                              _ints([40, 1], cuda_device), _ints([0, 1, 2], cuda_device))
    assert (out == 0).all()
    # No request at all, rows of padding only.
    for pages in (0, 2):
        cache = torch.zeros((pages, 16, 2, 64), dtype=torch.bfloat16, device=cuda_device)
        out, lse = ops.paged_attention(
            rows(3, 4), cache, cache, torch.zeros((0, 3), dtype=torch.int32, device=cuda_device),
            _ints([], cuda_device), _ints([0], cuda_device), return_lse=True)
        assert (out == 0).all() and (lse == -math.inf).all()
    cache = torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    out = ops.paged_attention(rows(2, 4), cache, cache,
                              torch.zeros((2, 0), dtype=torch.int32, device=cuda_device),
                              _ints([40, 1], cuda_device), _ints([0, 1, 2], cuda_device))
    assert (out == 0).all()


def test_strides(cuda_device):
    """Operands as views: one projection's Q, K and V, head-major storage, a
    cache with the heads outside the pages' rows, an output inside a larger one."""
    lens = [37, 1, 100]
    total = sum(lens)
    fused = _rows((total, 4 + 2 + 2, 128), torch.bfloat16, 31, cuda_device)
    q, k, v = fused.split((4, 2, 2), dim=1)
    starts = _starts(lens, cuda_device)
    base = ops.packed_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts)
    assert torch.equal(base, ops.packed_attention(q, k, v, starts))
    heads_first = [x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v)]
    holder = torch.zeros((total, 6, 160), dtype=torch.bfloat16, device=cuda_device)
    out = holder[:, 1:5, 16:144]
    ops.packed_attention(*heads_first, starts, out=out)
    assert torch.equal(out, base)
    assert (holder[:, 0] == 0).all() and (holder[:, :, :16] == 0).all()
    # An odd head stride is copied, not refused.
    odd = torch.zeros((total, 4, 129), dtype=torch.bfloat16, device=cuda_device)
    odd[..., :128] = q
    assert torch.equal(base, ops.packed_attention(odd[..., :128], k, v, starts))
    kv_lens = [60, 7]
    k_cache, v_cache, table = _cache(kv_lens, 16, 2, 128, torch.bfloat16, 32, cuda_device)
    args = (_ints(table, cuda_device), _ints(kv_lens, cuda_device), _ints([0, 1, 2], cuda_device))
    base = ops.paged_attention(q[:2], k_cache, v_cache, *args)
    kh = k_cache.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    both = torch.stack((v_cache, v_cache), dim=1)[:, 1]
    wide_table = torch.full((2, 50), 99, dtype=torch.int32, device=cuda_device)
    wide_table[:, :args[0].shape[1]] = args[0]
    assert torch.equal(base, ops.paged_attention(q[:2], kh, both,
                                                 wide_table[:, :args[0].shape[1]], *args[1:]))


def test_scale(cuda_device):
    q = _rows((70, 2, 64), torch.bfloat16, 33, cuda_device)
    k = _rows((70, 2, 64), torch.bfloat16, 34, cuda_device)
    v = _rows((70, 2, 64), torch.bfloat16, 35, cuda_device)
    out, lse = ops.packed_attention(q, k, v, _starts([70], cuda_device), scale=0.31,
                                    return_lse=True)
    _check(out, lse, oracle.packed(q, k, v, [70], scale=0.31), 64, 70, v.abs().max().item())


def test_cache_past_32_bits(cuda_device):
    """A cache of more than 2^32 bytes and 2^31 elements: pages at its far end."""
    pages, page, kh, dim = 9000, 256, 8, 128  # 4.7 GB, 2.36e9 elements
    k_cache = torch.zeros((pages, page, kh, dim), dtype=torch.bfloat16, device=cuda_device)
    v_cache = torch.zeros_like(k_cache)
    own = [8999, 0, 8750, 8200]
    q_lens, kv_lens = [1, 60], [400, 512]
    for i, p in enumerate(own):
        k_cache[p] = _rows((page, kh, dim), torch.bfloat16, 36 + i, cuda_device)
        v_cache[p] = _rows((page, kh, dim), torch.bfloat16, 40 + i, cuda_device)
    table = [own[:2], own[2:]]
    for lens in (q_lens, [1, 1]):
        q = _rows((sum(lens), kh, dim), torch.bfloat16, 44, cuda_device)
        out, lse = ops.paged_attention(q, k_cache, v_cache, _ints(table, cuda_device),
                                       _ints(kv_lens, cuda_device), _starts(lens, cuda_device),
                                       return_lse=True)
        _check(out, lse, oracle.paged(q, k_cache, v_cache, table, kv_lens, lens), dim, 512,
               v_cache[own].abs().max().item())
    new = _rows((3, kh, dim), torch.bfloat16, 45, cuda_device)
    slots = torch.tensor([pages * page - 1, -1, 8500 * page + 17], device=cuda_device)
    ops.paged_write(new, new + 1, k_cache, v_cache, slots)
    assert torch.equal(k_cache[-1, -1], new[0]) and torch.equal(v_cache[8500, 17], new[2] + 1)
    assert (k_cache[8500, 16] == 0).all() and (k_cache[8500, 18] == 0).all()


def test_repeats_bit_for_bit(cuda_device):
    kv_lens, q_lens = [5000, 800, 33, 2100], [1, 1, 1, 1]
    k_cache, v_cache, table = _cache(kv_lens, 16, 2, 128, torch.bfloat16, 46, cuda_device)
    q = _rows((200, 8, 128), torch.bfloat16, 47, cuda_device)
    for lens in (q_lens, [30, 100, 3, 67]):
        args = (q[:sum(lens)], k_cache, v_cache, _ints(table, cuda_device),
                _ints(kv_lens, cuda_device), _starts(lens, cuda_device))
        first = ops.paged_attention(*args, return_lse=True)
        for _ in range(5):
            again = ops.paged_attention(*args, return_lse=True)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ---------------------------------------------------------------------------
# Plan and write
# ---------------------------------------------------------------------------

def _run_plan(cached, new, table, free, page, tokens, device):
    held = torch.tensor(table, dtype=torch.int32, device=device)
    if not table:
        held = torch.zeros((0, 4), dtype=torch.int32, device=device)
    got = ops.paged_plan(_ints(cached, device), _ints(new, device), held, _ints(free, device),
                         page, tokens)
    return (got.q_start.tolist(), got.kv_lens.tolist(), got.slots.tolist(), got.status.tolist(),
            held.tolist())


@pytest.mark.parametrize("case", range(40))
def test_plan_against_oracle(cuda_device, case):
    """Random steps, among them empty ones, short free lists and short rows."""
    g = torch.Generator().manual_seed(case)

    def rand(lo, hi):
        return int(torch.randint(lo, hi + 1, (), generator=g))

    page = (16, 32, 128)[case % 3]
    requests = (0, 1, 7, 64, 513, 1500)[case % 6]
    longest = (1, 20, 300)[rand(0, 2)]
    cached = [rand(0, 400) for _ in range(requests)]
    new = [rand(0, longest) for _ in range(requests)]
    if requests > 3:
        cached[1], new[2] = -4, -9  # negative lengths count as 0
    need = [-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(cached, new)]
    width = max(need + [1]) - (1 if case % 5 == 4 else 0)
    free = torch.randperm(sum(need) + 5, generator=g).tolist()
    if case % 4 == 3:
        free = free[:max(0, len(free) // 3)]
    table = [[rand(0, 10 ** 6) for _ in range(width)] for _ in range(requests)]
    total = sum(max(n, 0) for n in new)
    tokens = total + (0, 13)[case % 2] if case % 7 else max(0, total - 5)
    if requests == 0 or width == 0:
        table = [[] for _ in range(requests)]
    got = _run_plan(cached, new, table, free, page, tokens, cuda_device)
    expected = oracle.plan(cached, new, table, free, page, tokens)
    for name, a, b in zip(("q_start", "kv_lens", "slots", "status", "table"), got, expected):
        assert a == b, name


def test_plan_most_requests_and_again(cuda_device):
    requests = 8192
    cached = _ints([i % 50 for i in range(requests)], cuda_device)
    new = _ints([1] * requests, cuda_device)
    table = torch.zeros((requests, 5), dtype=torch.int32, device=cuda_device)
    free = torch.arange(100, 100 + requests, dtype=torch.int32, device=cuda_device)
    plan = ops.paged_plan(cached, new, table, free, 16, requests)
    expected = oracle.plan(cached.tolist(), new.tolist(), [[0] * 5] * requests, free.tolist(), 16,
                           requests)
    assert plan.slots.tolist() == expected[2] and table.tolist() == expected[4]
    assert plan.status.tolist() == expected[3]
    before = table.clone()
    again = ops.paged_plan(cached, new, table, free, 16, requests)
    assert torch.equal(before, table)
    assert all(torch.equal(a, b) for a, b in zip(plan, again))
    with pytest.raises(ValueError, match="8192"):
        ops.paged_plan(_ints([0] * 8193, cuda_device), _ints([0] * 8193, cuda_device),
                       torch.zeros((8193, 1), dtype=torch.int32, device=cuda_device), free, 16, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 8), (63, 5, 40), (700, 8, 128), (257, 3, 64)])
def test_write(cuda_device, dtype, tokens, heads, dim):
    page, pages = 16, 60
    g = torch.Generator().manual_seed(50)
    slots = torch.randperm(page * pages, generator=g)[:tokens]
    slots[::7] = torch.tensor([-1, page * pages, 2 ** 40, -2 ** 62])[torch.arange(
        slots[::7].numel()) % 4]
    kv = _rows((tokens, 2 * heads, dim), torch.float32, 51, cuda_device).to(dtype)
    k, v = kv[:, :heads], kv[:, heads:]
    k_cache = _rows((pages, page, heads, dim), torch.float32, 52, cuda_device).to(dtype)
    v_cache = torch.zeros((pages, heads, page, dim), dtype=dtype, device=cuda_device).transpose(1, 2)
    want_k, want_v = k_cache.clone(), v_cache.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < page * pages:
            want_k[s // page, s % page] = k[t]
            want_v[s // page, s % page] = v[t]
    ops.paged_write(k, v, k_cache, v_cache, slots.to(cuda_device))
    assert torch.equal(k_cache, want_k) and torch.equal(v_cache, want_v)


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------

def test_prompt_chunks_and_steps_as_one_prompt(cuda_device):
    """Prompts, then a chunk, then single tokens through plan, write and paged
    attention give what the whole sequences give at once."""
    kh, h, dim, page = 2, 8, 128, 16
    steps = [[37, 5, 0, 210], [64, 1, 30, 3], [1, 1, 1, 1], [1, 0, 1, 1], [1, 1, 0, 1]]
    whole = [sum(s[r] for s in steps) for r in range(4)]
    g = torch.Generator().manual_seed(60)
    q, k, v = ([torch.randn((n, heads, dim), generator=g).to(torch.bfloat16).to(cuda_device)
                for n in whole] for heads in (h, kh, kh))
    pages = 60
    k_cache = torch.full((pages, page, kh, dim), math.nan, dtype=torch.bfloat16,
                         device=cuda_device)
    v_cache = k_cache.clone()
    table = torch.full((4, 20), -1, dtype=torch.int32, device=cuda_device)
    free = torch.randperm(pages, generator=g).to(torch.int32).to(cuda_device)
    cached = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    done, parts = [0] * 4, [[] for _ in range(4)]
    for new in steps:
        pick = [slice(d, d + n) for d, n in zip(done, new)]
        qs, ks, vs = (torch.cat([x[r][pick[r]] for r in range(4)]) for x in (q, k, v))
        plan = ops.paged_plan(cached, _ints(new, cuda_device), table, free, page, sum(new) + 3)
        padded = [torch.cat((x, x[:1].expand(3, -1, -1))) for x in (qs, ks, vs)]
        ops.paged_write(padded[1], padded[2], k_cache, v_cache, plan.slots)
        out = ops.paged_attention(padded[0], k_cache, v_cache, table, plan.kv_lens, plan.q_start)
        assert (out[sum(new):] == 0).all()
        for r, part in enumerate(out[:sum(new)].split(new)):
            parts[r].append(part)
        taken, lost = plan.status.tolist()
        assert lost == 0
        free, cached = free[taken:], plan.kv_lens
        done = [d + n for d, n in zip(done, new)]
    got = torch.cat([torch.cat(p) for p in parts])
    allq, allk, allv = (torch.cat(x) for x in (q, k, v))
    expected = oracle.packed(allq, allk, allv, whole)
    _check(got, None, expected, dim, max(whole), allv.abs().max().item())
    at_once, lse = ops.packed_attention(allq, allk, allv, _starts(whole, cuda_device),
                                        return_lse=True)
    _check(at_once, lse, expected, dim, max(whole), allv.abs().max().item())


def test_captured_step_replays_with_new_lengths(cuda_device):
    """A decoding step captured once (plan, write, attention) and replayed as the
    requests grow, eager steps of another cache between the replays."""
    kh, h, dim, page, requests, pages = 2, 8, 64, 16, 5, 64

    def caches():
        g = torch.Generator().manual_seed(70)
        k = torch.randn((pages, page, kh, dim), generator=g).to(torch.bfloat16).to(cuda_device)
        return {"k": k, "v": k.flip(0).contiguous(),
                "table": torch.arange(requests * 8, dtype=torch.int32,
                                      device=cuda_device).view(requests, 8).clone(),
                "free": torch.arange(40, 64, dtype=torch.int32, device=cuda_device),
                "cached": _ints([3, 0, 100, 47, 16], cuda_device)}

    new = _ints([1] * requests, cuda_device)
    q, k, v = (torch.empty((requests, n, dim), dtype=torch.bfloat16, device=cuda_device)
               for n in (h, kh, kh))

    def step(s):
        plan = ops.paged_plan(s["cached"], new, s["table"], s["free"], page, requests)
        ops.paged_write(k, v, s["k"], s["v"], plan.slots)
        out, lse = ops.paged_attention(q, s["k"], s["v"], s["table"], plan.kv_lens, plan.q_start,
                                       return_lse=True)
        s["cached"].copy_(plan.kv_lens)
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
    for i in range(6):
        inputs(i)
        graph.replay()
        got = [t.clone() for t in held]
        torch.cuda.synchronize()
        expected = step(eager)
        assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1]), i
        for name in ("k", "v", "table", "cached"):
            assert torch.equal(eager[name], captured[name]), (i, name)


def test_calls_on_two_streams(cuda_device):
    """Calls that overlap on two streams keep their workspaces apart."""
    kv_lens, q_lens = [9000, 500, 4000], [1, 1, 1]
    k_cache, v_cache, table = _cache(kv_lens, 16, 2, 128, torch.bfloat16, 80, cuda_device)
    q = _rows((3, 8, 128), torch.bfloat16, 81, cuda_device)
    args = (k_cache, v_cache, _ints(table, cuda_device), _ints(kv_lens, cuda_device),
            _starts(q_lens, cuda_device))
    expected = [ops.paged_attention(q * s, *args) for s in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    inputs = [q * 1, q * 2]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append(ops.paged_attention(inputs[i], *args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(r, expected[i]) for r in results[i])


def test_two_captured_graphs_replayed_in_turn(cuda_device):
    """Two graphs of calls that split their keys, replayed alternately with eager
    calls between: neither disturbs the other's results."""
    kv_lens = [6000, 300]
    k_cache, v_cache, table = _cache(kv_lens, 16, 2, 128, torch.bfloat16, 90, cuda_device)
    at = (k_cache, v_cache, _ints(table, cuda_device), _ints(kv_lens, cuda_device))
    q = [_rows((n, 8, 128), torch.bfloat16, 91 + n, cuda_device) for n in (2, 90)]
    starts = [_starts([1, 1], cuda_device), _starts([60, 30], cuda_device)]
    expected = [ops.paged_attention(x, *at, s) for x, s in zip(q, starts)]
    graphs, outs = [], []
    for x, s in zip(q, starts):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.paged_attention(x, *at, s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.paged_attention(x, *at, s))
        graphs.append(graph)
    for i in range(6):
        graphs[i % 2].replay()
        ops.paged_attention(q[1], *at, starts[1])
        graphs[1 - i % 2].replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, expected):
            assert torch.equal(out, want), i


@pytest.mark.parametrize("requests", [65, 1025, 3000])
def test_many_requests(cuda_device, requests):
    """More requests than one wave, one workgroup or the list's LDS holds; some
    bring nothing, some have no keys."""
    g = torch.Generator().manual_seed(requests)
    kv_lens = torch.randint(0, 60, (requests,), generator=g).tolist()
    q_lens = [int(i % 7 != 3) for i in range(requests)]
    k_cache, v_cache, table = _cache(kv_lens, 16, 1, 64, torch.bfloat16, 92, cuda_device)
    q = _rows((sum(q_lens), 4, 64), torch.bfloat16, 93, cuda_device)
    out, lse = ops.paged_attention(q, k_cache, v_cache, _ints(table, cuda_device),
                                   _ints(kv_lens, cuda_device), _starts(q_lens, cuda_device),
                                   return_lse=True)
    _check(out, lse, oracle.paged(q, k_cache, v_cache, table, kv_lens, q_lens), 64, 60,
           v_cache[~v_cache.isnan()].abs().max().item())
    # Their prompts, packed: 128-row tiles, several requests of none.
    lens = [n * (1 + i % 3) for i, n in enumerate(q_lens)]
    total = sum(lens)
    q, k, v = (_rows((total, h, 64), torch.bfloat16, 94 + h, cuda_device) for h in (20, 1, 1))
    out = ops.packed_attention(q, k, v, _starts(lens, cuda_device))
    _check(out, None, oracle.packed(q, k, v, lens), 64, 3, v.abs().max().item())


@pytest.mark.parametrize("requests", [7, 70])
@pytest.mark.parametrize("heads", [(6, 3, 80), (12, 12, 96), (5, 5, 40), (4, 2, 128)], ids=str)
def test_steps_of_heads_in_shared_lines(cuda_device, requests, heads):
    """Decoding steps whose key heads share memory lines, with and without the list;
    whole and cut keys.  (128 dims share lines when the cache starts inside one.)"""
    h, kh, dim = heads
    g = torch.Generator().manual_seed(requests)
    kv_lens = torch.randint(0, 400, (requests,), generator=g).tolist()
    kv_lens[1], kv_lens[5] = 4000, 2500
    k_cache, v_cache, table = _cache(kv_lens, 16, kh, dim, torch.bfloat16, 101, cuda_device)
    if dim == 128:
        store = torch.empty(k_cache.numel() + 8, dtype=k_cache.dtype, device=cuda_device)
        k_cache = store[8:].view(k_cache.shape).copy_(k_cache)
        assert k_cache.data_ptr() % 128 == 16
    q_lens = [1 + (i % 5 == 2) for i in range(requests)]
    q = _rows((sum(q_lens), h, dim), torch.bfloat16, 102, cuda_device)
    out, lse = ops.paged_attention(q, k_cache, v_cache, _ints(table, cuda_device),
                                   _ints(kv_lens, cuda_device), _starts(q_lens, cuda_device),
                                   return_lse=True)
    _check(out, lse, oracle.paged(q, k_cache, v_cache, table, kv_lens, q_lens), dim, 4000,
           v_cache[~v_cache.isnan()].abs().max().item())


def test_tail_and_long_tiles_are_cut(cuda_device):
    """Calls of more than one round of 128-row tiles: equal tiles whose last round
    is cut, one tile far longer than its share, ragged ones that stay whole."""
    g = torch.Generator().manual_seed(95)
    for q_lens, k_lens, heads in (
            ([128] * 50, [512] * 50, 12),        # 600 equal tiles: 88 of them are cut
            ([128] * 129, [130] * 128 + [6000], 4),  # one long
            (torch.randint(1, 400, (60,), generator=g).tolist(), None, 8)):
        k_lens = k_lens or q_lens
        q = _rows((sum(q_lens), heads, 64), torch.bfloat16, 96, cuda_device)
        k = _rows((sum(k_lens), heads, 64), torch.bfloat16, 97, cuda_device)
        v = _rows((sum(k_lens), heads, 64), torch.bfloat16, 98, cuda_device)
        out, lse = ops.packed_attention(q, k, v, _starts(q_lens, cuda_device),
                                        _starts(k_lens, cuda_device), causal=False,
                                        return_lse=True)
        _check(out, lse, oracle.packed(q, k, v, q_lens, k_lens, causal=False), 64, max(k_lens),
               v.abs().max().item())


def test_shared_pages_and_output_over_q(cuda_device):
    """Requests that share a prefix's pages, and an output that takes q's place."""
    k_cache, v_cache, table = _cache([64, 40], 16, 2, 64, torch.bfloat16, 99, cuda_device)
    table[1][:2] = table[0][:2]
    q = _rows((30, 4, 64), torch.bfloat16, 100, cuda_device)
    args = (k_cache, v_cache, _ints(table, cuda_device), _ints([64, 40], cuda_device),
            _ints([0, 10, 30], cuda_device))
    out = ops.paged_attention(q, *args)
    _check(out, None, oracle.paged(q, k_cache, v_cache, table, [64, 40], [10, 20]), 64, 64,
           v_cache[~v_cache.isnan()].abs().max().item())
    assert ops.paged_attention(q, *args, out=q) is q
    assert torch.equal(q, out)


def test_refusals(cuda_device):
    def rows(n, h, d=64, t=torch.bfloat16):
        return torch.zeros((n, h, d), dtype=t, device=cuda_device)

    starts = _ints([0, 4], cuda_device)
    q, k = rows(4, 4), rows(4, 2)
    with pytest.raises(ValueError, match="float32"):
        ops.packed_attention(rows(4, 4, t=torch.float32), rows(4, 2, t=torch.float32),
                             rows(4, 2, t=torch.float32), starts)
    with pytest.raises(ValueError, match="like q"):
        ops.packed_attention(q, k.half(), k, starts)
    with pytest.raises(ValueError, match="share"):
        ops.packed_attention(rows(4, 5), k, k, starts)
    with pytest.raises(ValueError, match="head dimension"):
        ops.packed_attention(q, rows(4, 2, 72), rows(4, 2, 72), starts)
    with pytest.raises(ValueError, match="head_dim"):
        ops.packed_attention(rows(4, 4, 136), rows(4, 2, 136), rows(4, 2, 136), starts)
    with pytest.raises(ValueError, match="head_dim"):
        ops.packed_attention(rows(4, 4, 60), rows(4, 2, 60), rows(4, 2, 60), starts)
    with pytest.raises(ValueError, match="int32"):
        ops.packed_attention(q, k, k, starts.long())
    with pytest.raises(ValueError, match="one value more"):
        ops.packed_attention(q, k, k, starts[:0])
    with pytest.raises(ValueError, match="k_start"):
        ops.packed_attention(q, k, k, starts, _ints([0, 1, 2], cuda_device))
    with pytest.raises(ValueError, match="scale"):
        ops.packed_attention(q, k, k, starts, scale=-0.5)
    with pytest.raises(ValueError, match="out"):
        ops.packed_attention(q, k, k, starts, out=torch.zeros_like(k))
    with pytest.raises(ValueError, match="expanded"):
        ops.packed_attention(q, k, k, starts, out=q[:1].expand(4, -1, -1))
    with pytest.raises(ValueError, match="aligned"):
        ops.packed_attention(q, k, k, starts, out=rows(4, 4, 66)[..., :64])
    with pytest.raises(ValueError, match="rows, heads, head_dim"):
        ops.packed_attention(q[0], k, k, starts)
    cache = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    table, lens = torch.zeros((1, 2), dtype=torch.int32, device=cuda_device), starts[1:]
    odd = torch.zeros((3, 24, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError, match="page_size"):
        ops.paged_attention(q, odd, odd, table, lens, starts)
    with pytest.raises(ValueError, match="block_table"):
        ops.paged_attention(q, cache, cache, table.expand(2, -1), lens, starts)
    with pytest.raises(ValueError, match="block_table"):
        ops.paged_attention(q, cache, cache, table.long(), lens, starts)
    with pytest.raises(ValueError, match="kv_lens"):
        ops.paged_attention(q, cache, cache, table, lens.long(), starts)
    with pytest.raises(ValueError, match="q_start"):
        ops.paged_attention(q, cache, cache, table, lens, starts[:1])
    with pytest.raises(ValueError, match="k_cache"):
        ops.paged_attention(q, cache[..., ::2], cache[..., ::2], table, lens, starts)
    with pytest.raises(ValueError, match="k_cache"):
        ops.paged_attention(q, cache.half(), cache, table, lens, starts)
    with pytest.raises(ValueError, match="shape"):
        ops.paged_attention(q, cache, cache[:2], table, lens, starts)
    slots = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    with pytest.raises(ValueError, match="slots"):
        ops.paged_write(k, k, cache, cache.clone(), slots.int())
    with pytest.raises(ValueError, match="expanded"):
        ops.paged_write(k, k, cache[:1].expand(3, -1, -1, -1), cache, slots)
    with pytest.raises(ValueError, match="agree"):
        ops.paged_write(rows(4, 3), rows(4, 3), cache, cache.clone(), slots)
    with pytest.raises(ValueError, match="2 or 4 bytes"):
        ops.paged_write(k.double(), k.double(), cache.double(), cache.double(), slots)
    with pytest.raises(ValueError, match="16-byte"):
        ops.paged_write(rows(4, 2, 12), rows(4, 2, 12), cache[..., :12].contiguous(),
                        cache[..., :12].contiguous(), slots)
    with pytest.raises(ValueError, match="new"):
        ops.paged_plan(lens, starts, table, starts, 16, 4)
    with pytest.raises(ValueError, match="tokens"):
        ops.paged_plan(lens, lens, table, starts, 16, -1)
    with pytest.raises(ValueError, match="page_size"):
        ops.paged_plan(lens, lens, table, starts, 20, 4)


def test_axes_of_one_entry(cuda_device):
    """An axis of one entry may have any stride."""
    base = _rows((7, 3, 64), torch.bfloat16, 101, cuda_device)
    one = torch.as_strided(base, (1, 2, 64), (13, 64, 1))
    out = ops.packed_attention(one, one, one, _ints([0, 1], cuda_device))
    assert torch.equal(out, one)
    single = torch.as_strided(base, (7, 1, 64), (192, 5, 1))
    expected = oracle.packed(single, single, single, [7])
    out = ops.packed_attention(single, single, single, _ints([0, 7], cuda_device))
    _check(out, None, expected, 64, 7, single.abs().max().item())
