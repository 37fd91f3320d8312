"""Rotated cache writes and the 4-bit cache without a GPU: the oracles against plain
definitions, the host-side argument checks of the C entry points (which run before any
HIP call), and the rejection of CPU tensors."""

import ctypes
import math

import pytest
import torch

from dit_sparse_atten_amd import _lib, ops
from oracle import fp4 as oracle

FAKE = ctypes.c_void_p(4096)  # never dereferenced: the checks come first
ODD = ctypes.c_void_p(4104)


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIBRARY_PATH.exists():
        pytest.skip("libdsa.so not built")
    return _lib.load()


# ---------------------------------------------------------------------------
# Oracles
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("halves", [False, True])
def test_rotate_oracle_is_a_complex_product(halves):
    g = torch.Generator().manual_seed(0)
    x = torch.randn((5, 3, 24), generator=g, dtype=torch.float64)
    angle = torch.randn((7, 8), generator=g, dtype=torch.float64)
    cos_sin = torch.stack((angle.cos(), angle.sin()), -1)
    positions = torch.tensor([6, 0, 3, -1, 7])
    got = oracle.rotate(x, positions, cos_sin, halves)
    pairs = x[..., :16].reshape(5, 3, 2, 8).transpose(2, 3) if halves else \
        x[..., :16].reshape(5, 3, 8, 2)
    z = torch.view_as_complex(pairs.contiguous())
    turned = z[:3] * torch.polar(torch.ones(3, 8, dtype=torch.float64),
                                 angle[positions[:3]])[:, None]
    parts = torch.view_as_real(turned)
    want = parts.transpose(2, 3).reshape(3, 3, 16) if halves else parts.reshape(3, 3, 16)
    torch.testing.assert_close(got[:3, :, :16], want, rtol=1e-12, atol=1e-12)
    assert torch.equal(got[..., 16:], x[..., 16:]) and torch.equal(got[3:], x[3:])


def test_nearest_oracle():
    """Every value is the nearest of the group's, its exponent the smallest that holds the
    largest element times 7."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn((300, 2, 40), generator=g) * torch.exp2(
        torch.randint(-20, 20, (300, 2, 1), generator=g).float())
    got = oracle.nearest(x, torch.bfloat16)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    grid = torch.cat((-grid.flip(0), grid))
    for part, values in ((x[..., :32], got[..., :32]), (x[..., 32:], got[..., 32:])):
        top = part.double().abs().amax(-1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(top / 7)))
        nearest = (part.double()[..., None] / scale[..., None] - grid).abs().amin(-1) * scale
        torch.testing.assert_close((values - part).abs(), nearest, rtol=1e-12, atol=0)
        assert (values.abs() <= 6 * scale).all()
    ties = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] * 4])
    assert oracle.nearest(ties, torch.bfloat16)[0, :8].tolist() == [0, 1, 1, 2, 2, 4, 4, 6]
    # fp16's exponents end at 13 and -23.
    assert oracle.nearest(torch.full((1, 32), 65504.0), torch.float16)[0, 0] == 6 * 2.0 ** 13
    assert oracle.nearest(torch.full((1, 32), 2.0 ** -24), torch.float16)[0, 0] == 2.0 ** -24
    odd = torch.ones((3, 40))
    odd[0, 3], odd[1, 39] = math.inf, math.nan
    got = oracle.nearest(odd, torch.bfloat16)
    assert got[0, :32].isnan().all() and (got[0, 32:] == 1).all() and got[1, 32:].isnan().all()


def test_decode_oracle():
    """The bytes' places: element 2 i in the low half, scales behind the codes."""
    cache = torch.zeros((2, 3, 16, 72), dtype=torch.uint8)
    flat = cache.view(2, 3, -1)
    flat[1, 2, 5 * 32 + 1] = 0xB3          # keys, row 5: dims 2 and 3
    flat[1, 2, 16 * 32 + 7 * 32 + 16] = 0x7F  # values, row 7: dims 32 and 33
    flat[1, 2, 2 * 16 * 32:] = 127
    flat[1, 2, 2 * 16 * 32 + 4 * 5] = 129
    flat[1, 2, 2 * 16 * 32 + 64 + 4 * 7 + 1] = 126
    k, v = oracle.decode(cache, 64)
    assert k.shape == (2, 16, 3, 64)
    assert k[1, 5, 2, :5].tolist() == [0, 0, 6, -6, 0] and (k != 0).sum() == 2
    assert v[1, 7, 2, 32:35].tolist() == [-3, 3, 0] and (v != 0).sum() == 2


# ---------------------------------------------------------------------------
# C entry points
# ---------------------------------------------------------------------------

def _rotary(lib, **change):
    args = dict(q=FAKE, q_out=FAKE, k=FAKE, v=FAKE, k_cache=FAKE, v_cache=FAKE, dtype=0,
                strides=_lib.int64_array([64] * 14), tokens=4, heads=4, kv_heads=2, head_dim=64,
                rot_dim=32, halves=0, pages=3, page_size=16, slots=FAKE, positions=FAKE,
                cos_sin=FAKE, max_positions=9, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_paged_write_rotary(*args.values())


def _fp4(lib, **change):
    args = dict(q=FAKE, q_out=FAKE, k=FAKE, v=FAKE, cache=FAKE, dtype=0,
                strides=_lib.int64_array([64] * 8 + [4096, 1152]), tokens=4, heads=4, kv_heads=2,
                head_dim=64, rot_dim=32, halves=0, pages=3, page_size=16, slots=FAKE,
                positions=FAKE, cos_sin=FAKE, max_positions=9, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_paged_write_fp4(*args.values())


def _read(lib, **change):
    args = dict(cache=FAKE, strides=_lib.int64_array([4096, 1152]), k=FAKE, v=FAKE, dtype=0,
                pages=3, page_size=16, kv_heads=2, head_dim=64, list=FAKE, count=2, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_paged_read_fp4(*args.values())


def _attend(lib, **change):
    args = dict(q=FAKE, cache=FAKE, o=FAKE, dtype=0,
                strides=_lib.int64_array([64, 64, 4096, 1152, 64, 64]), q_rows=4, requests=2,
                heads=4, kv_heads=2, head_dim=64, pages=3, page_size=16, table=FAKE,
                table_stride=4, table_width=4, kv_lens=FAKE, q_start=FAKE, scale=0.1, causal=1,
                fill=1, lse=None, workspace=FAKE, workspace_bytes=1 << 30, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_paged_attention_fp4(*args.values())


SHARED = [
    ("tokens", -1, "size", _lib.DSA_EINVAL), ("heads", -1, "size", _lib.DSA_EINVAL),
    ("kv_heads", 0, "size", _lib.DSA_EINVAL), ("pages", -1, "size", _lib.DSA_EINVAL),
    ("max_positions", -1, "size", _lib.DSA_EINVAL), ("strides", None, "strides", _lib.DSA_EINVAL),
    ("dtype", 2, "dtype", _lib.DSA_EUNSUPPORTED), ("dtype", 7, "dtype", _lib.DSA_EUNSUPPORTED),
    ("head_dim", 136, "head_dim", _lib.DSA_EUNSUPPORTED),
    ("head_dim", 60, "head_dim", _lib.DSA_EUNSUPPORTED),
    ("head_dim", 0, "head_dim", _lib.DSA_EUNSUPPORTED),
    ("rot_dim", 8, "rot_dim", _lib.DSA_EUNSUPPORTED),
    ("rot_dim", 80, "rot_dim", _lib.DSA_EUNSUPPORTED),
    ("rot_dim", -16, "rot_dim", _lib.DSA_EUNSUPPORTED), ("halves", 2, "halves", _lib.DSA_EINVAL),
    ("page_size", 24, "page_size", _lib.DSA_EUNSUPPORTED),
    ("page_size", 8, "page_size", _lib.DSA_EUNSUPPORTED),
    ("heads", 5000, "heads", _lib.DSA_EUNSUPPORTED),
    ("kv_heads", 5000, "heads", _lib.DSA_EUNSUPPORTED),
    ("q", ODD, "aligned", _lib.DSA_EINVAL), ("q_out", ODD, "aligned", _lib.DSA_EINVAL),
    ("k", ODD, "aligned", _lib.DSA_EINVAL), ("v", ODD, "aligned", _lib.DSA_EINVAL),
    ("cos_sin", ODD, "aligned", _lib.DSA_EINVAL),
    *[(name, None, "null", _lib.DSA_EINVAL)
      for name in ("q", "q_out", "k", "v", "slots", "positions", "cos_sin")],
]


@pytest.mark.parametrize("call", [_rotary, _fp4], ids=["rotary", "fp4"])
@pytest.mark.parametrize("name,value,text,status", SHARED)
def test_write_refusals(lib, call, name, value, text, status):
    assert call(lib, **{name: value}) == status
    assert text in _lib.last_error()


def test_cache_refusals(lib):
    for name in ("k_cache", "v_cache"):
        for bad in (None, ODD):
            assert _rotary(lib, **{name: bad}) == _lib.DSA_EINVAL
    for call in (_fp4, _read, _attend):
        for bad in (None, ODD):
            assert call(lib, cache=bad) == _lib.DSA_EINVAL
        assert call(lib, page_size=1 << 21) == _lib.DSA_EUNSUPPORTED
        assert "page_size" in _lib.last_error()
        assert call(lib, page_size=40) == _lib.DSA_EUNSUPPORTED
    for call, count, at in ((_rotary, 14, ()), (_fp4, 10, (8, 9)), (_read, 2, (0, 1)),
                            (_attend, 6, (2, 3))):
        for i in range(count):
            for bad in (-64, 1156 if i in at else 60):
                strides = [4096 if j in at else 64 for j in range(count)]
                strides[i] = bad
                assert call(lib, strides=_lib.int64_array(strides)) == _lib.DSA_EINVAL, (call, i)
                assert "strides" in _lib.last_error()


@pytest.mark.parametrize("name,value,text", [
    ("strides", None, "strides"), ("pages", -1, "size"), ("kv_heads", 0, "size"),
    ("count", -1, "size"), ("dtype", 2, "dtype"), ("head_dim", 132, "head_dim"),
    ("k", None, "null"), ("v", None, "null"), ("k", ODD, "aligned"),
])
def test_read_refusals(lib, name, value, text):
    assert _read(lib, **{name: value}) < 0
    assert text in _lib.last_error()
    assert _read(lib, list=None, count=4) == _lib.DSA_EINVAL  # of three pages


@pytest.mark.parametrize("name,value,text", [
    ("strides", None, "strides"), ("q", None, "null"), ("o", None, "null"),
    ("q_start", None, "null"), ("kv_lens", None, "lengths"), ("table", None, "block table"),
    ("dtype", 2, "dtype"), ("heads", 5, "share"), ("kv_heads", 0, "share"),
    ("head_dim", 136, "head_dim"), ("head_dim", 12, "head_dim"), ("q_rows", -1, "negative"),
    ("requests", -1, "negative"), ("pages", -1, "page count"), ("table_width", -1, "table"),
    ("table_stride", 3, "table"), ("scale", 0.0, "scale"), ("scale", math.inf, "scale"),
    ("scale", math.nan, "scale"), ("scale", 3e38, "scale"), ("causal", 2, "causal"),
    ("fill", 2, "fill"), ("q", ODD, "aligned"), ("workspace", None, "workspace"),
    ("workspace", ODD, "aligned"), ("workspace_bytes", 256, "workspace"),
])
def test_attention_refusals(lib, name, value, text):
    assert _attend(lib, **{name: value}) < 0
    assert text in _lib.last_error()


def test_workspace_sizes(lib):
    """As over 16-bit pages; 16-row tiles up to 32 rows a request, or 64 where they leave
    compute units idle, 512 workgroups for them instead of 256 where they are more, whole
    tiles up to 2,048 keys."""
    size = lib.dsa_paged_attention_fp4_workspace_bytes

    def expected(rows, requests, heads, kv, dim, keys):
        group = heads // kv
        narrow = rows * group <= 32 * requests or (
            rows * group <= 64 * requests and rows * heads <= 4096)
        many = narrow and max(requests, rows * group // 16) * kv > 256
        tile, slots, uncut = (16, 512 if many else 256, 2048) if narrow else (128, 512, 640)
        tiles = max(1, rows * group // tile + requests)
        cut = keys > uncut and slots >= kv
        partials = 2 * slots // kv if cut else 0
        splits = min(tiles, partials // 2)
        at = 256 + (2048 if many else 1024) + ((requests + 1) * 4 + 255) // 256 * 256
        at += (tiles + partials) * 64 + (splits * 64 + 255) // 256 * 256
        return at + partials * kv * tile * ((64 if dim <= 64 else 128) + 2) * 4

    for case in ((8, 2, 4, 2, 64, 100), (32, 32, 64, 8, 128, 16384), (33, 33, 64, 8, 128, 16384),
                 (512, 512, 64, 8, 64, 1000), (300, 300, 4, 1, 40, 5000), (2, 2, 600, 600, 64, 2000),
                 (2, 2, 300, 300, 64, 2100), (4, 4, 32, 8, 128, 2048), (4, 4, 32, 8, 128, 2049),
                 (128, 32, 64, 8, 128, 9000), (129, 32, 64, 8, 128, 9000), (64, 4, 32, 8, 128, 9000),
                 (65, 4, 32, 8, 128, 9000), (128, 16, 64, 8, 128, 9000), (32, 2, 32, 2, 64, 9000),
                 (2500, 40, 32, 8, 128, 30000), (5, 0, 1, 1, 8, 0)):
        assert size(*case) == expected(*case), case
    for bad in ((0, 1, 1, 1, 64, 9), (1, -1, 1, 1, 64, 9), (1, 1, 3, 2, 64, 9), (1, 1, 1, 0, 64, 9),
                (1, 1, 1, 1, 0, 9), (1, 1, 1, 1, 64, -1)):
        assert size(*bad) == 0, bad


def test_nothing_to_do_is_no_call(lib):
    assert _rotary(lib, tokens=0) == _lib.DSA_OK
    assert _fp4(lib, tokens=0) == _lib.DSA_OK
    assert _read(lib, count=0) == _lib.DSA_OK
    assert _attend(lib, q_rows=0, workspace=None, workspace_bytes=0) == _lib.DSA_OK


def test_cpu_tensors_are_rejected():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    ints, slots = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int64)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    packed = ops.paged_cache_fp4(2, 16, 2, 64, "cpu")
    assert packed.shape == (2, 2, 16, 72) and packed.dtype == torch.uint8
    angles = torch.zeros(3, 16, 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_write_rotary(q, q, cache, cache, slots, ints, angles)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_write_fp4(q, q, packed, slots)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_read_fp4(packed, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention_fp4(q, packed, torch.zeros((2, 4), dtype=torch.int32), ints[:2], ints)


@pytest.mark.parametrize("args,match", [
    ((2, 24, 2, 64), "page_size"), ((2, 8, 2, 64), "page_size"), ((2, 1 << 21, 2, 64), "page_size"),
    ((2, 16, 2, 136), "head_dim"), ((2, 16, 2, 4), "head_dim"), ((-1, 16, 2, 64), "pages"),
    ((2, 16, 0, 64), "heads"),
])
def test_cache_shapes(args, match):
    with pytest.raises(ValueError, match=match):
        ops.paged_cache_fp4(*args, "cpu")
