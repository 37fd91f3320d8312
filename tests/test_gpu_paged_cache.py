"""The paged key/value cache on the GPU where it can go wrong: rows of one 16-byte
chunk."""

import pytest
import torch

from dit_sparse_atten_amd import ops

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
