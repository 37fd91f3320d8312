"""Values that are not finite in sequences of different lengths: rows that see them
have them, other rows do not, and a call that meets them stays near its time.

Tolerance of finite elements: the probabilities' rounding to the input type and the
result's, half a step each, of sum_j p_j |v_j|, in fp16 also 2^-25 max|v| a key for
probabilities below its smallest normal one; 2^-10 for everything in fp32 (128 products
a score of magnitudes up to 16, twice, 2^-12; up to 5,000 terms a sum, twice, 2^-10.7)."""

import math

import pytest
import torch

from dit_sparse_atten_amd import ops
from oracle import sequences as oracle

pytestmark = pytest.mark.gpu

VALUES = (math.inf, -math.inf, math.nan)


def _starts(lens, device):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=device)


def _rows(shape, dtype, seed, device):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(device)


def _compare(got, expected, v_max, keys):
    out, _, weight, reach = expected
    got = got.cpu()
    seen = ~torch.isfinite(out)
    assert torch.equal(got[seen].isnan(), out[seen].isnan())
    assert torch.equal(got[seen].nan_to_num(0, 1, -1).double(), out[seen].nan_to_num(0, 1, -1))
    assert reach.max() <= 16 and keys <= 5000
    step = torch.finfo(got.dtype).eps / 2
    bound = (2 * step + 2 ** -10) * weight[~seen]
    if got.dtype == torch.float16:
        bound = bound + keys * 2.0 ** -25 * v_max + 2.0 ** -25
    error = (got[~seen].double() - out[~seen]).abs()
    assert torch.isfinite(error).all(), "a hidden value reached a row"
    assert (error <= bound + 1e-30).all(), (error / bound).max()


CALLS = [
    ([150], [150]),              # a prompt
    ([70, 40], [3000, 200]),     # chunks, long keys cut into parts
    ([3, 1, 2], [900, 33, 2500]),  # few rows of each: 16-row tiles
    ([16], [5000]),
    ([40, 3], [30, 1]),          # rows without a key
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("heads", [(4, 4, 128), (8, 2, 128), (4, 1, 64), (3, 3, 96), (6, 2, 40)],
                         ids=str)
@pytest.mark.parametrize("q_lens,k_lens", CALLS, ids=str)
@pytest.mark.parametrize("where", ["early", "last rows", "all over"])
def test_values_that_are_not_finite(cuda_device, dtype, heads, q_lens, k_lens, where):
    h, kh, dim = heads
    q = _rows((sum(q_lens), h, dim), dtype, 1, cuda_device)
    k = _rows((sum(k_lens), kh, dim), dtype, 2, cuda_device)
    v = _rows((sum(k_lens), kh, dim), dtype, 3, cuda_device)
    starts = _starts(q_lens, cuda_device), _starts(k_lens, cuda_device)
    clean, stat = ops.packed_attention(q, k, v, *starts, return_lse=True)
    v_max = v.abs().max().item()
    at = 0
    for n, m in zip(q_lens, k_lens):
        hits = {"early": [0, 5], "last rows": [m - n // 2, m - 1, m - n // 3],
                "all over": range(0, m, 37)}[where]
        for i, hit in enumerate(hits):
            if 0 <= hit < m:
                # A dimension of every seven, so that most stay finite.
                v[at + hit, :, i % 7::7] = VALUES[i % 3]
                if i % 2:
                    v[at + hit, :, (i + 3) % 7::14] = VALUES[(i + 1) % 3]
        at += m
    expected = oracle.packed(q, k, v, q_lens, k_lens)
    out, lse = ops.packed_attention(q, k, v, *starts, return_lse=True)
    assert torch.equal(lse, stat)
    _compare(out, expected, v_max, max(k_lens))
    # The same keys in pages, the rows behind them not finite either.
    page = 16
    need = [-(-m // page) for m in k_lens]
    pages, width = sum(need), max(need) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(4)).tolist()
    kc = torch.full((pages, page, kh, dim), math.nan, dtype=dtype, device=cuda_device)
    vc = torch.full_like(kc, math.inf)
    table, at = [], 0
    for m, count in zip(k_lens, need):
        own = [order.pop() for _ in range(count)]
        table.append(own + [-1] * (width - count))
        for i, p in enumerate(own):
            rows = min(page, m - i * page)
            kc[p, :rows] = k[at + i * page:at + i * page + rows]
            vc[p, :rows] = v[at + i * page:at + i * page + rows]
        at += m

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=cuda_device)

    paged = ops.paged_attention(q, kc, vc, ints(table), ints(k_lens), starts[0])
    _compare(paged, expected, v_max, max(k_lens))
    paged = ops.paged_attention(q, kc, vc, ints(table), ints(k_lens), starts[0], causal=False)
    _compare(paged, oracle.packed(q, k, v, q_lens, k_lens, causal=False), v_max, max(k_lens))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [128, 96, 64])
@pytest.mark.parametrize("stride", [0, 8])
@pytest.mark.parametrize("n,m", [(1, 1), (40, 1), (1, 5), (3, 37), (60, 70), (16, 2000),
                                 (150, 1500)], ids=str)
def test_infinite_values_of_rows_that_overlap(cuda_device, n, m, stride, dim, causal):
    """One key (an axis of one entry), and V whose tokens share memory: expanded, or 8
    elements apart.  What the rows see is infinite, nothing turns to NaN."""
    q = _rows((n, 4, dim), torch.bfloat16, 8, cuda_device)
    k = _rows((m, 2, dim), torch.bfloat16, 9, cuda_device)
    store = _rows((2 * dim + 8 * m,), torch.bfloat16, 10, cuda_device)
    # (in rows 8 elements apart, the last ones alone reach the store's end)
    store[3], store[-dim - 8] = math.inf, -math.inf
    v = torch.as_strided(store, (m, 2, dim), (stride, dim, 1))
    starts = _starts([n], cuda_device), _starts([m], cuda_device)
    out = ops.packed_attention(q, k, v, *starts, causal=causal)
    expected = oracle.packed(q, k, v.contiguous(), [n], [m], causal)
    _compare(out, expected, 5.0, m)
    # Packed in pages, every row of a page the same one.
    pages = -(-m // 16)
    kc = torch.full((pages * 16, 2, dim), math.nan, dtype=k.dtype, device=cuda_device)
    kc[:m] = k
    vc = torch.as_strided(store, (pages, 16, 2, dim), (0, 0, dim, 1))
    table = torch.arange(pages, dtype=torch.int32, device=cuda_device)[None]
    out = ops.paged_attention(q, kc.view(pages, 16, 2, dim), vc, table, starts[1][1:], starts[0],
                              causal=causal)
    expected = oracle.packed(q, k, vc.reshape(-1, 2, dim)[:m], [n], [m], causal)
    _compare(out, expected, 5.0, m)


def _time(call):
    best = math.inf
    for _ in range(5):
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        call()
        end.record()
        end.synchronize()
        best = min(best, begin.elapsed_time(end))
    return best


@pytest.mark.parametrize("n,m,heads", [(4096, 4096, (4, 2)), (16, 60000, (1, 1))], ids=str)
def test_time_of_values_that_are_not_finite(cuda_device, n, m, heads):
    """One infinite value that nearly every row sees costs next to nothing, and values
    in every row's last keys, where each wave has to tell who sees them, a few times
    the call at most."""
    h, kh = heads
    q = _rows((n, h, 128), torch.bfloat16, 5, cuda_device)
    k = _rows((m, kh, 128), torch.bfloat16, 6, cuda_device)
    v = _rows((m, kh, 128), torch.bfloat16, 7, cuda_device)
    starts = _starts([n], cuda_device), _starts([m], cuda_device)

    def call():
        ops.packed_attention(q, k, v, *starts)

    call()
    clean = _time(call)
    v[5] = math.inf
    early = _time(call)
    v[::16, :, ::2] = math.nan
    v[1::16] = -math.inf
    all_over = _time(call)
    print(f"{n} x {m}: {clean:.3f} ms, early {early:.3f}, all over {all_over:.3f}", flush=True)
    assert early <= 2 * clean and all_over <= 10 * clean
