"""Scores over a 4-bit cache are sums in fp32 of exact products, whatever the dims'
magnitudes: against the float64 oracle of the values that the cache stands for.

Tolerances as for the 16-bit cache: a score of D products is off by at most D 2^-24 of its
sum of magnitudes S, the LSE by that and m 2^-24 + 2^-18 + 2^-22 |LSE| (sums of m terms,
exponential and logarithm, the units' change), the probabilities by twice the score's error;
they are rounded to the input type (half a step, eps / 2) before they meet V and the result
once more.  In fp16 a probability below 2^-14 of the row's reference is off by 2^-25 of it
at most, and a result by 2^-25."""

import math

import pytest
import torch

from dit_sparse_atten_amd import ops
from oracle import fp4 as oracle_fp4
from oracle import sequences as oracle

pytestmark = pytest.mark.gpu


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _starts(lens, device):
    return _ints([sum(lens[:i]) for i in range(len(lens) + 1)], device)


def _check(got, lse, expected, dim, keys, v_max):
    out, stat, weight, reach = expected
    step = torch.finfo(got.dtype).eps / 2
    score = dim * 2.0 ** -24 * reach
    fp32 = (torch.expm1(2 * score).t() + 2.0 * keys * 2.0 ** -24 + 2.0 ** -18)[..., None]
    bound = (step + fp32) * weight * (1 + step) + step * out.abs() + 1e-30
    if got.dtype == torch.float16:
        bound = bound + keys * 2.0 ** -25 * v_max + 2.0 ** -25
    error = (got.double().cpu() - out).abs()
    limit = score + keys * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -22 * stat.abs()
    off = (lse.double().cpu() - stat).abs()
    assert torch.isfinite(error).all() and torch.isfinite(off).all()
    assert (off <= limit).all(), f"LSE off by {(off / limit).max().item():.3f} bounds"
    assert (error <= bound).all(), f"error {(error / bound).max().item():.3f} times its bound"


def _queries(kind, shape, g):
    q = torch.randn(shape, generator=g)
    dim = shape[-1]
    if kind == "outlier dims":  # as turned keys and queries have: one among its neighbours
        q[..., 5] *= 60
        q[..., dim - 3] *= 100
    elif kind == "every magnitude":
        q *= torch.exp2(torch.randint(-9, 6, shape, generator=g).float())
    elif kind == "one large":
        q *= 2.0 ** -11
        q[..., dim // 2] = 15.0
    return q


CALLS = {
    "steps": ([1] * 6, [1, 2, 16, 700, 3000, 0]),
    "a few tokens": ([4, 9], [4, 400]),
    "prompts": ([150, 3], [150, 3]),
    "chunks": ([70, 130], [900, 2000]),
    "a few rows of a 128-row tile": ([140], [140]),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("kind", ["normal", "outlier dims", "every magnitude", "one large"])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (3, 3, 96), (4, 2, 40), (2, 1, 8)],
                         ids=str)
@pytest.mark.parametrize("call", CALLS)
def test_scores(cuda_device, call, heads, kind, dtype):
    q_lens, kv_lens = CALLS[call]
    h, kh, dim = heads
    page, g = 16, torch.Generator().manual_seed(dim)
    q = _queries(kind, (sum(q_lens), h, dim), g).to(dtype).to(cuda_device)
    need = [-(-m // page) for m in kv_lens]
    cache = ops.paged_cache_fp4(sum(need) + 1, page, kh, dim, cuda_device)
    table, slots, at = [], [], 0
    for m, pages in zip(kv_lens, need):
        table.append([at + i for i in range(pages)] + [-1] * (max(need) - pages))
        slots.append(torch.arange(m) + at * page)
        at += pages
    # Keys of groups of different magnitudes, none of a group's elements at 0.
    k, v = (torch.randn((sum(kv_lens), kh, dim), generator=g) for _ in range(2))
    k += 0.3 * k.sign()
    k *= torch.exp2(torch.randint(-3, 3, (sum(kv_lens), kh, -(-dim // 32)), generator=g).float()
                    ).repeat_interleave(32, -1)[..., :dim]
    ops.paged_write_fp4(k.to(dtype).to(cuda_device), v.to(dtype).to(cuda_device), cache,
                        torch.cat(slots).to(cuda_device))
    held = oracle_fp4.decode(cache, dim)
    out, lse = ops.paged_attention_fp4(
        q, cache, _ints(table, cuda_device), _ints(kv_lens, cuda_device),
        _starts(q_lens, cuda_device), scale=0.25 / math.sqrt(dim), return_lse=True)
    expected = oracle.paged(q, *held, table, kv_lens, q_lens, True, 0.25 / math.sqrt(dim))
    empty = expected[1] == -math.inf
    assert (lse.cpu()[empty] == -math.inf).all()
    lse, stat = lse.cpu().masked_fill(empty, 0), expected[1].masked_fill(empty, 0)
    _check(out, lse, (expected[0], stat, *expected[2:]), dim, max(kv_lens),
           held[1].abs().max().item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("dim", [128, 40])
def test_keys_of_the_smallest_and_largest_exponents(cuda_device, dim, n, dtype):
    """Elements down to the type's smallest numbers against the largest queries, and the
    other way round: every product enters."""
    m, page = 200, 16
    g = torch.Generator().manual_seed(n)
    low, high = oracle_fp4.EXPONENTS[dtype]
    q = torch.randn((n, 2, dim), generator=g)
    k = torch.randint(-6, 7, (m, 2, dim), generator=g).float()
    k[..., ::32] = 6  # (so that the group's exponent is the intended one)
    big = (q * 2.0 ** (high - 2), k * 2.0 ** low)
    small = (q * 2.0 ** (low + 12), k * 2.0 ** high)
    v = torch.randn((m, 2, dim), generator=g).to(dtype)
    for q, k in (big, small):
        q, k = q.to(dtype).to(cuda_device), k.to(dtype).to(cuda_device)
        assert q.isfinite().all() and k.isfinite().all()
        cache = ops.paged_cache_fp4(-(-m // page), page, 2, dim, cuda_device)
        ops.paged_write_fp4(k, v.to(cuda_device), cache, torch.arange(m, device=cuda_device))
        held = oracle_fp4.decode(cache, dim)
        table = [list(range(-(-m // page)))]
        reach = (q.double().cpu().abs().amax() * held[0].abs().amax()).item() * dim
        scale = 20 / reach
        out, lse = ops.paged_attention_fp4(q, cache, _ints(table, cuda_device),
                                           _ints([m], cuda_device), _ints([0, n], cuda_device),
                                           scale=scale, return_lse=True)
        expected = oracle.paged(q, *held, table, [m], [n], True, scale)
        _check(out, lse, expected, dim, m, held[1].abs().max().item())
