"""Attention over a 4-bit cache in each of its launches: items listed by the schedule kernel
or worked out by the workgroups, whole and cut tiles, one round of them and more, one
workgroup of eight waves or two of four.  `_plan` says which one a call takes, from the same
rule as the host's, and is held against the workspace's size, so that no case slips into
another launch unseen.  Tolerances: `test_gpu_paged_fp4._check` with sums in fp32."""

import pytest
import torch

from dit_sparse_atten_amd import _lib, ops
from test_gpu_paged_fp4 import DTYPES, _Cache, _check, _rows, _starts

pytestmark = pytest.mark.gpu


def _plan(rows, requests, heads, kv, dim, keys):
    """(16-row tiles, two workgroups a compute unit, cut, listed) of a call."""
    group = heads // kv
    total = rows * group
    narrow = total <= 32 * requests or (total <= 64 * requests and total * kv <= 4096)
    pairs = narrow and max(requests, total // 16) * kv > 256
    height, slots = (16, 512 if pairs else 256) if narrow else (128, 512)
    tiles = max(1, total // height + requests)
    cut = keys > (2048 if narrow else 640) and slots >= kv
    listed = not (requests <= 64 and tiles <= 64 and tiles * kv <= (256 if narrow else 512)
                  and (narrow or tiles * kv * min(keys, 1 << 30) <= 80 * slots * 64))
    partials = 2 * slots // kv if cut else 0
    at = 256 + (2048 if pairs else 1024) + ((requests + 1) * 4 + 255) // 256 * 256
    at += (tiles + partials) * 64 + (min(tiles, partials // 2) * 64 + 255) // 256 * 256
    at += partials * kv * height * ((64 if dim <= 64 else 128) + 2) * 4
    size = _lib.load().dsa_paged_attention_fp4_workspace_bytes
    assert size(rows, requests, heads, kv, dim, keys) == at, "the rule has changed"
    return narrow, pairs, cut, listed


def _lens(seed, count, low, high):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, high + 1, (count,), generator=g).tolist()


def _run(device, heads, q_lens, kv_lens, dtype, causal, plan, page=16, seed=80):
    h, kh, dim = heads
    cache = _Cache(kv_lens, page, kh, dim, seed, device)
    keys = len(cache.table[0]) * page
    assert _plan(sum(q_lens), len(q_lens), h, kh, dim, keys) == plan
    q = _rows((sum(q_lens), h, dim), DTYPES[dtype], seed + 1, device)
    args = (q, *cache.args(device), _starts(q_lens, device))
    out, lse = ops.paged_attention_fp4(*args, causal=causal, return_lse=True)
    _check(out, lse, cache.expected(q, q_lens, causal), dim, max(kv_lens), cache.v_max(), 0.0)
    again = ops.paged_attention_fp4(*args, causal=causal, return_lse=True)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [128, 96, 64, 40])
@pytest.mark.parametrize("heads,count,causal", [
    ((8, 4), 70, True),      # more tiles than run at a time, tails cut
    ((4, 2), 70, False),     # one round, cut as it takes
    ((10, 10), 66, False),   # more than eight key heads
], ids=str)
def test_128_row_tiles_listed_and_cut(cuda_device, dtype, dim, heads, count, causal):
    q_lens = _lens(1, count, 30, 150)
    kv_lens = [n + more for n, more in zip(q_lens, _lens(2, count, 0, 300))]
    kv_lens[3], kv_lens[10], q_lens[20] = 2000, q_lens[10] // 2, 0
    q_lens[5] = 300
    _run(cuda_device, (*heads, dim), q_lens, kv_lens, dtype, causal, (False, False, True, True))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads", [(9, 9, 96), (6, 2, 64), (16, 4, 128)], ids=str)
def test_128_row_tiles_listed_and_whole(cuda_device, dtype, heads):
    q_lens = _lens(3, 80, 40, 140)
    kv_lens = [max(0, n + more) for n, more in zip(q_lens, _lens(4, 80, -60, 400))]
    _run(cuda_device, heads, q_lens, kv_lens, dtype, True, (False, False, False, True))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,q_lens,kv_lens,causal", [
    # 30 tiles x 8 key heads on 256 compute units, some cut
    ((16, 8, 128), [1] * 30, [6000, 4000, 2300] + _lens(5, 27, 0, 400), True),
    ((16, 8, 64), [1] * 30, [6000, 4000, 2300] + _lens(5, 27, 0, 400), False),
    # up to three tiles of a request
    ((16, 1, 40), [3, 1, 2, 0] * 16 + [3], [5000, 9000] + _lens(6, 63, 0, 300), True),
    ((40, 20, 96), [2] * 12, [3000] + _lens(7, 11, 0, 500), True),
], ids=["30 x 8", "30 x 8, 64 dims", "65 requests", "20 key heads"])
def test_16_row_tiles_listed_and_cut(cuda_device, dtype, heads, q_lens, kv_lens, causal):
    _run(cuda_device, heads, q_lens, kv_lens, dtype, causal, (True, False, True, True))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_16_row_tiles_listed_and_whole(cuda_device, dtype):
    _run(cuda_device, (16, 8, 128), [1] * 31, _lens(8, 31, 0, 1900), dtype, True,
         (True, False, False, True))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("kv_lens,cut", [([3000] + [40] * 79, True), ([1500] + [40] * 79, False)],
                         ids=["cut", "whole"])
def test_16_row_tiles_in_pairs(cuda_device, dtype, kv_lens, cut):
    """Steps of many requests, and of more rows than one tile holds."""
    _run(cuda_device, (8, 4, 128), [1] * 80, kv_lens, dtype, True, (True, True, cut, True))
    _run(cuda_device, (32, 4, 64), [3, 4, 0, 5] * 20, kv_lens, dtype, True,
         (True, True, cut, True))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,q_lens,kv_lens,plan", [
    ((8, 2, 128), [1] * 4, [700, 0, 2000, 5], (True, False, False, False)),
    ((8, 2, 64), [1] * 4, [7000, 0, 2100, 5], (True, False, True, False)),
    ((8, 2, 96), [130, 40], [500, 600], (False, False, False, False)),
    ((8, 2, 128), [130, 40], [900, 3000], (False, False, True, False)),
], ids=str)
def test_unlisted(cuda_device, dtype, heads, q_lens, kv_lens, plan):
    _run(cuda_device, heads, q_lens, kv_lens, dtype, True, plan)
