"""A value that is not a number reaches every row that sees its key, also where another wave
or part of the tile holds scores so much larger that its own weight goes to 0.

The keys are zeros but for a few, one element each, against queries of one element: scores
of 0, and of 384 (2^553 times the weight, past what fp32 tells from 0).  Rows that see none
of the large scores weigh their keys alike, the others have the large keys' mean.  Finite
elements: the probabilities' rounding and the result's, half a step each, of sum_j p_j |v_j|,
and (m + 2^6) 2^-24 for up to m terms of the sums, exponentials and joins."""

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


# (tokens, keys) of each request, (query heads, key heads, dim)
CALLS = {
    "a whole 16-row tile": ([1], [700], (8, 2, 128)),
    "a whole 16-row tile, 64 dims": ([2, 1], [900, 1100], (4, 2, 64)),
    "a few parts": ([1], [2500], (4, 2, 128)),
    "a few rows, a few parts": ([3, 2], [4000, 3000], (4, 1, 96)),
    "many parts": ([1], [60000], (2, 1, 128)),
    "many parts of two requests": ([1, 4], [40000, 50000], (4, 2, 64)),
    "two workgroups a compute unit": ([1] * 300, [6000] + [90] * 299, (4, 1, 128)),
    "128-row tiles, the last by pairs of waves": ([150], [170], (2, 2, 128)),
    "by pairs of waves, 96 dims": ([40], [700], (4, 1, 96)),
    "128-row tiles, cut": ([70], [3000], (4, 2, 128)),
    "128-row tiles, cut often": ([100], [30000], (1, 1, 64)),
}


def _places(m):
    """(the key whose value is not a number, the large keys)."""
    yield 5, [40, m - 2]                     # another half of a 64-key step, another part
    yield 70, [5, 150]                       # another wave
    yield m - 3, [m // 2, 3]
    yield m // 2 + 17, [m // 3]


def _close(got, expected, keys):
    out, _, weight, _ = expected
    got = got.double().cpu()
    assert torch.equal(got.isnan(), out.isnan()), (got.isnan() ^ out.isnan()).nonzero()[:5]
    finite = ~out.isnan()
    step = torch.finfo(torch.bfloat16).eps / 2
    bound = (2 * step + step * step + (keys + 64) * 2.0 ** -24) * weight.nan_to_num(0) + 1e-30
    assert ((got - out).abs()[finite] <= bound[finite]).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("call", CALLS)
def test_value_of_no_weight(cuda_device, call, causal):
    q_lens, kv_lens, (h, kh, dim) = CALLS[call]
    page, tokens = 16, sum(kv_lens)
    q = torch.zeros((sum(q_lens), h, dim), dtype=torch.bfloat16, device=cuda_device)
    q[..., 0] = 1
    need = [-(-m // page) for m in kv_lens]
    table, slots, at = [], [], 0
    for m, pages in zip(kv_lens, need):
        table.append([at + i for i in range(pages)] + [-1] * (max(need) - pages))
        slots.append(torch.arange(m) + at * page)
        at += pages
    slots = torch.cat(slots).to(cuda_device)
    rest = (_ints(table, cuda_device), _ints(kv_lens, cuda_device), _starts(q_lens, cuda_device))
    g = torch.Generator().manual_seed(1)
    values = torch.randn((tokens, kh, dim), generator=g).to(torch.bfloat16)
    cache = ops.paged_cache_fp4(at, page, kh, dim, cuda_device)
    held = [torch.zeros((at, page, kh, dim), dtype=torch.bfloat16, device=cuda_device)
            for _ in range(2)]
    for i, (hit, large) in enumerate(_places(kv_lens[0])):
        group = i % -(-dim // 32)
        k, v = torch.zeros_like(values), values.clone()
        k[large, :, 0] = 384.0
        v[hit, :, 32 * group + 3] = math.nan
        args = (k.to(cuda_device), v.to(cuda_device))
        ops.paged_write_fp4(*args, cache, slots)
        own = oracle_fp4.nearest(v.float(), torch.bfloat16)
        out = ops.paged_attention_fp4(q, cache, *rest, causal=causal, scale=1.0)
        _close(out, oracle.packed(q, k, own, q_lens, kv_lens, causal, 1.0), max(kv_lens))
        # The 16-bit cache, whose joins are the same: the element itself.
        ops.paged_write(*args, *held, slots)
        out = ops.paged_attention(q, *held, *rest, causal=causal, scale=1.0)
        expected = oracle.packed(q, k, v, q_lens, kv_lens, causal, 1.0)
        _close(out, expected, max(kv_lens))
        held[1][held[1].isnan()] = math.inf
        again = ops.paged_attention(q, *held, *rest, causal=causal, scale=1.0)
        seen = expected[0].isnan().to(cuda_device)
        assert not again[seen].isfinite().any() and torch.equal(again[~seen], out[~seen])
