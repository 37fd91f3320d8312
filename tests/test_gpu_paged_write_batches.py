"""Large writes, whose workgroups walk several heads: the same bits as the same tokens
written a slice at a time, where every workgroup has one head (the form that the oracles
check).  And reads of more than the caches hold, against reads of a few pages each."""

import pytest
import torch

from dit_sparse_atten_amd import ops

pytestmark = pytest.mark.gpu

# tokens, heads, key heads, dim, turned dims
CASES = [
    (16384, 12, 5, 128, 128),   # eight heads a workgroup, 4 of 12 and 5 left
    (16384, 13, 3, 128, 96),
    (9000, 12, 5, 96, 64),
    (19001, 7, 2, 80, 32),
    (4100, 13, 3, 128, 0),
    (40000, 3, 9, 40, 32),
    (60000, 9, 1, 16, 16),
]


def _batch(tokens, heads, kv_heads, rows):
    """Heads of a workgroup of `rows` tokens."""
    return min(8, max(1, -(-tokens // rows) * (heads + 2 * kv_heads) // 1024))


def _rows(dim, fp4):
    return 256 // (4 * -(-dim // 32)) if fp4 else 256 // ((dim // 8 + 1) // 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("fp4", [False, True], ids=["16 bits", "4 bits"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_heads_of_a_batch(cuda_device, case, fp4, halves, dtype):
    tokens, heads, kv_heads, dim, rot = case
    page, rows = 16, _rows(dim, fp4)
    assert _batch(tokens, heads, kv_heads, rows) > 1
    slice_of = max(rows, 1500 // (heads + 2 * kv_heads) * rows)
    assert _batch(slice_of, heads, kv_heads, rows) == 1
    g = torch.Generator(cuda_device).manual_seed(tokens)

    def random(*shape):
        return torch.randn(shape, generator=g, device=cuda_device)

    x = random(tokens, heads + 2 * kv_heads + 1, dim).to(dtype)
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:-1]
    angle = random(50, rot // 2).double() * 10
    cos_sin = torch.stack((angle.cos(), angle.sin()), -1).float()
    positions = torch.randint(-2, 52, (tokens,), generator=g, device=cuda_device,
                              dtype=torch.int32)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=g, device=cuda_device)[:tokens]
    slots[::11] = -1
    if fp4:
        clean = [torch.randint(0, 250, (pages, kv_heads, page, 32 * -(-dim // 32) + 8),
                               generator=g, dtype=torch.uint8, device=cuda_device)]
    else:
        clean = [random(pages, page, kv_heads, dim).to(dtype) for _ in range(2)]

    def write(held, part, **more):
        call = ops.paged_write_fp4 if fp4 else ops.paged_write_rotary
        return call(k[part], v[part], *held, slots[part], positions[part], cos_sin, halves=halves,
                    **more)

    slices = [slice(a, min(a + slice_of, tokens)) for a in range(0, tokens, slice_of)]
    want = [c.clone() for c in clean]
    turned = torch.cat([write(want, part, q=q[part]) for part in slices])
    got = [c.clone() for c in clean]
    whole = write(got, slice(0, tokens), q=q)
    assert bool((whole == turned).all())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # In place, within the projection's rows, and without queries.
    own, again = x.clone(), [c.clone() for c in clean]
    view = own[:, :heads]
    assert write(again, slice(0, tokens), q=view, q_out=view) is view
    assert bool((view == turned).all()) and torch.equal(own[:, heads:], x[:, heads:])
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    again = [c.clone() for c in clean]
    assert write(again, slice(0, tokens)) is None
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("pages,page,kv_heads,dim", [(1700, 32, 8, 128), (3000, 16, 13, 96),
                                                     (700, 128, 15, 40), (140, 1024, 24, 16)])
def test_large_reads(cuda_device, pages, page, kv_heads, dim, dtype):
    assert pages * page * kv_heads * dim * 4 >= 192 << 20
    g = torch.Generator(cuda_device).manual_seed(dim)
    cache = torch.randint(0, 256, (pages, kv_heads, page, 32 * -(-dim // 32) + 8), generator=g,
                          dtype=torch.uint8, device=cuda_device)
    listed = torch.randperm(pages, generator=g, device=cuda_device).int()
    listed[5], listed[pages // 2] = -1, pages
    few = max(1, (64 << 20) // (page * kv_heads * dim * 4))
    for pages_of in (None, listed):
        got = ops.paged_read_fp4(cache, dim, pages_of, dtype)
        order = torch.arange(pages, device=cuda_device).int() if pages_of is None else pages_of
        for a in range(0, pages, few):
            part = ops.paged_read_fp4(cache, dim, order[a:a + few], dtype)
            for x, y in zip(got, part):
                torch.testing.assert_close(x[a:a + few], y, rtol=0, atol=0, equal_nan=True)
