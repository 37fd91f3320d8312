"""Queries of one type over a cache written from the other, and over exponents that no write
makes: values are what a read of the cache in the queries' type gives, or not a number.

Tolerances as for the 16-bit cache: the probabilities' rounding to the input type and the
result's, half a step (eps / 2) each, of sum_j p_j |v_j|; fp32: a score's D products 2 D
2^-24 of its sum of magnitudes, m 2^-23 for sums of m terms, 2^-18 for the exponentials and
joins; in fp16 2^-25 max|v| for probabilities below its normal ones, a key, and 2^-25."""

import pytest
import torch

from dit_sparse_atten_amd import ops
from oracle import sequences as oracle

pytestmark = pytest.mark.gpu


def _ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _close(got, expected, dim, keys, v_max, seen):
    out, _, weight, reach = expected
    step = torch.finfo(got.dtype).eps / 2
    fp32 = (2 * dim * 2.0 ** -24 * reach.t() + 2 * keys * 2.0 ** -24 + 2.0 ** -18)[..., None]
    bound = (step + fp32) * weight * (1 + step) + step * out.abs() + 1e-30
    if got.dtype == torch.float16:
        bound = bound + keys * 2.0 ** -25 * v_max + 2.0 ** -25
    error = (got.double().cpu() - out).abs()
    assert (error <= bound)[~seen].all()


@pytest.mark.parametrize("n,m", [(1, 700), (4, 900), (150, 170), (70, 3000)])
@pytest.mark.parametrize("heads", [(4, 2, 128), (2, 1, 40)], ids=str)
@pytest.mark.parametrize("dtype,exponent", [
    (torch.float16, 13), (torch.float16, 14), (torch.float16, 15), (torch.float16, 60),
    (torch.bfloat16, 125), (torch.bfloat16, 126), (torch.bfloat16, 127)], ids=str)
def test_values_of_large_exponents(cuda_device, dtype, exponent, heads, n, m):
    """Past the type's largest exponent a group's dims are NaN in the rows that see its key,
    and no other row knows of it."""
    h, kh, dim = heads
    page, groups = 16, -(-dim // 32)
    pages = -(-m // page)
    g = torch.Generator().manual_seed(3)
    q = torch.randn((n, h, dim), generator=g).to(dtype).to(cuda_device)
    k, v = (torch.randn((m, kh, dim), generator=g).to(torch.bfloat16).to(cuda_device)
            for _ in range(2))
    cache = ops.paged_cache_fp4(pages, page, kh, dim, cuda_device)
    ops.paged_write_fp4(k, v, cache, torch.arange(m, device=cuda_device))
    hit, group = m - n + n // 2, groups - 1  # seen by the rows from n // 2 on
    at = 2 * page * 16 * groups + 4 * page + 4 * (hit % page) + group
    cache.view(pages, kh, -1)[hit // page, :, at] = exponent + 127
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    out = ops.paged_attention_fp4(q, cache, table, _ints([m], cuda_device),
                                  _ints([0, n], cuda_device))
    k16, v16 = (x.reshape(-1, kh, dim)[:m] for x in ops.paged_read_fp4(cache, dim, dtype=dtype))
    low, high = {torch.float16: (-23, 13), torch.bfloat16: (-125, 125)}[dtype]
    past = exponent > high
    seen = torch.zeros((n, h, dim), dtype=torch.bool)
    if past:
        seen[n // 2:, :, 32 * group:] = True
        assert out.isnan()[seen.to(cuda_device)].all()
        v16[hit] = v16[hit].nan_to_num(0, 0, 0)
        v16[hit, :, 32 * group:] = 0
    expected = oracle.packed(q, k16, v16, [n], [m])
    # The sums of p v are in fp32 before they are divided by the sum of p: m weights of up to
    # 2^8 (the reference follows the largest score from that far) times a row's mean |v|.
    large = expected[2] * m * 2.0 ** 8 > torch.finfo(torch.float32).max
    finite = torch.isfinite(out).cpu()
    assert finite[~seen & ~large].all(), "only those rows and dims"
    _close(out, expected, dim, m, v16.abs().max().item(), seen | large)


@pytest.mark.parametrize("n", [1, 100])
def test_the_other_type(cuda_device, n):
    """What a read in the queries' type gives, subnormal numbers among it."""
    m, dim, page = 600, 128, 16
    g = torch.Generator().manual_seed(4)
    k = torch.randn((m, 2, dim), generator=g)
    v = torch.randn((m, 2, dim), generator=g) * torch.exp2(
        torch.randint(-30, 12, (m, 2, 4), generator=g).float()).repeat_interleave(32, -1)
    for written, own in ((torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)):
        cache = ops.paged_cache_fp4(38, page, 2, dim, cuda_device)
        ops.paged_write_fp4(k.to(written).to(cuda_device), v.to(written).to(cuda_device), cache,
                            torch.arange(m, device=cuda_device))
        q = torch.randn((n, 4, dim), generator=g).to(own).to(cuda_device)
        table = torch.arange(38, dtype=torch.int32, device=cuda_device)[None]
        out = ops.paged_attention_fp4(q, cache, table, _ints([m], cuda_device),
                                      _ints([0, n], cuda_device))
        held = [x.reshape(-1, 2, dim)[:m] for x in ops.paged_read_fp4(cache, dim, dtype=own)]
        expected = oracle.packed(q, *held, [n], [m])
        _close(out, expected, dim, m, held[1].abs().max().item(),
               torch.zeros(out.shape, dtype=torch.bool))
