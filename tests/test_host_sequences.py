"""Sequence operators without a GPU: the oracles against plain definitions, the
host-side argument checks of the C entry points (which run before any HIP call),
workspace sizes, and the rejection of CPU tensors."""

import ctypes
import math

import pytest
import torch

from dit_sparse_atten_amd import _lib, ops
from oracle import sequences as oracle


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIBRARY_PATH.exists():
        pytest.skip("libdsa.so not built")
    return _lib.load()


# ---------------------------------------------------------------------------
# Oracles
# ---------------------------------------------------------------------------

def _dense(q, k, v, causal):
    """One sequence by the formula, every head with its own copy of its keys."""
    n, heads, dim = q.shape
    m = k.shape[0]
    k = k.repeat_interleave(heads // k.shape[1], dim=1).double()
    v = v.repeat_interleave(heads // v.shape[1], dim=1).double()
    s = torch.einsum("thd,jhd->htj", q.double(), k) * dim ** -0.5
    if causal:
        s = s.masked_fill(torch.arange(m)[None] > torch.arange(n)[:, None] + m - n, -math.inf)
    return torch.einsum("htj,jhd->thd", torch.softmax(s, -1), v), torch.logsumexp(s, -1)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,m", [(1, 1), (5, 5), (3, 9), (1, 20)])
def test_attend_oracle(causal, n, m):
    g = torch.Generator().manual_seed(n * 100 + m)
    q, k, v = (torch.randn((r, h, 16), generator=g) for r, h in ((n, 6), (m, 2), (m, 2)))
    out, lse, weight, reach = oracle.attend(q, k, v, causal)
    expected, stat = _dense(q, k, v, causal)
    torch.testing.assert_close(out, expected, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(lse, stat, rtol=1e-12, atol=1e-12)
    assert (weight >= out.abs() - 1e-12).all() and (reach > 0).all()


def test_attend_oracle_rows_without_keys():
    q, k, v = torch.randn(6, 2, 8), torch.randn(4, 2, 8), torch.randn(4, 2, 8)
    out, lse, _, _ = oracle.attend(q, k, v)
    assert (out[:2] == 0).all() and (lse[:, :2] == -math.inf).all()
    torch.testing.assert_close(out[2:], _dense(q[2:], k, v, True)[0], rtol=1e-12, atol=1e-12)
    out, lse, _, _ = oracle.attend(q, k, v, causal=False, present=torch.zeros(4, dtype=torch.bool))
    assert (out == 0).all() and (lse == -math.inf).all()


def test_paged_oracle_is_the_packed_one():
    g = torch.Generator().manual_seed(3)
    lens, q_lens, page = [20, 0, 33], [4, 0, 7], 16
    k = torch.randn((sum(lens), 2, 8), generator=g)
    v = torch.randn((sum(lens), 2, 8), generator=g)
    q = torch.randn((sum(q_lens), 4, 8), generator=g)
    table = [[4, 1, -1], [-1, -1, -1], [0, 5, 2]]
    k_cache, v_cache = torch.full((6, page, 2, 8), math.nan), torch.full((6, page, 2, 8), math.nan)
    at = 0
    for r, m in enumerate(lens):
        for j in range(m):
            k_cache[table[r][j // page], j % page] = k[at]
            v_cache[table[r][j // page], j % page] = v[at]
            at += 1
    packed = oracle.packed(q, k, v, q_lens, lens)
    paged = oracle.paged(q, k_cache, v_cache, table, lens, q_lens)
    for a, b in zip(packed, paged):
        torch.testing.assert_close(a, b, rtol=0, atol=0)
    # A page outside the cache leaves its keys out.
    table[2][1] = 77
    out = oracle.paged(q, k_cache, v_cache, table, lens, q_lens, causal=False)[0]
    rest = torch.cat((k[20:36], k[52:])), torch.cat((v[20:36], v[52:]))
    torch.testing.assert_close(out[4:], oracle.attend(q[4:], *rest, causal=False)[0], rtol=0,
                               atol=0)


def test_plan_oracle():
    table = [[7, -1, -1], [3, 4, -1], [-1, -1, -1]]
    got = oracle.plan([16, 20, 0], [1, 4, 17], table, [9, 8, 5], 16, 24)
    assert got[0] == [0, 1, 5, 22] and got[1] == [17, 24, 17]
    assert got[2] == ([9 * 16] + [4 * 16 + i for i in (4, 5, 6, 7)]
                      + [8 * 16 + i for i in range(16)] + [5 * 16] + [-1, -1])
    assert got[3] == [3, 0] and got[4] == [[7, 9, -1], [3, 4, -1], [8, 5, -1]]
    # One page short, and a slot map two tokens short of the last request.
    got = oracle.plan([16, 20, 0], [1, 4, 17], table, [9, 8], 16, 20)
    assert got[3] == [3, 2] and got[4][2] == [8, -1, -1] and len(got[2]) == 20


# ---------------------------------------------------------------------------
# Host checks
# ---------------------------------------------------------------------------

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def _packed(lib, **change):
    args = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, dtype=0, strides=_lib.int64_array([64] * 8),
                q_rows=8, k_rows=8, requests=2, heads=4, kv_heads=2, head_dim=64, q_start=FAKE,
                k_start=None, scale=0.1, causal=1, fill=1, lse=None, workspace=FAKE,
                workspace_bytes=1 << 30, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_packed_attention(*args.values())


def _paged(lib, **change):
    args = dict(q=FAKE, k_cache=FAKE, v_cache=FAKE, o=FAKE, dtype=0,
                strides=_lib.int64_array([64] * 10), q_rows=8, requests=2, heads=4, kv_heads=2,
                head_dim=64, pages=5, page_size=16, table=FAKE, table_stride=4, table_width=4,
                kv_lens=FAKE, q_start=FAKE, scale=0.1, causal=1, fill=1, lse=None,
                workspace=FAKE, workspace_bytes=1 << 30, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_paged_attention(*args.values())


SHARED = [
    ("q", None, "null", _lib.DSA_EINVAL),
    ("o", None, "null", _lib.DSA_EINVAL),
    ("q_start", None, "null", _lib.DSA_EINVAL),
    ("dtype", 2, "dtype", _lib.DSA_EUNSUPPORTED),
    ("heads", 5, "share", _lib.DSA_EINVAL),
    ("kv_heads", 0, "share", _lib.DSA_EINVAL),
    ("head_dim", 60, "head_dim", _lib.DSA_EUNSUPPORTED),
    ("head_dim", 136, "head_dim", _lib.DSA_EUNSUPPORTED),
    ("requests", -1, "negative", _lib.DSA_EINVAL),
    ("q_rows", -1, "negative", _lib.DSA_EINVAL),
    ("causal", 2, "causal", _lib.DSA_EINVAL),
    ("fill", 3, "fill", _lib.DSA_EINVAL),
    ("scale", 0.0, "scale", _lib.DSA_EINVAL),
    ("scale", -1.0, "scale", _lib.DSA_EINVAL),
    ("scale", math.inf, "scale", _lib.DSA_EINVAL),
    ("scale", math.nan, "scale", _lib.DSA_EINVAL),
    ("workspace", ctypes.c_void_p(4104), "aligned", _lib.DSA_EINVAL),
    ("o", ctypes.c_void_p(4098), "aligned", _lib.DSA_EINVAL),
    ("workspace_bytes", 100, "workspace", _lib.DSA_EINVAL),
    ("workspace", None, "workspace", _lib.DSA_EINVAL),
    ("strides", None, "strides", _lib.DSA_EINVAL),
]


@pytest.mark.parametrize("call", [_packed, _paged], ids=["packed", "paged"])
@pytest.mark.parametrize("name,value,text,status", SHARED)
def test_attention_refusals(lib, call, name, value, text, status):
    assert call(lib, **{name: value}) == status
    assert text in _lib.last_error()


def test_attention_stride_refusals(lib):
    for call, count in ((_packed, 8), (_paged, 10)):
        for i in range(count):
            for bad in (60, -64):
                strides = [64] * count
                strides[i] = bad
                assert call(lib, strides=_lib.int64_array(strides)) == _lib.DSA_EINVAL
                assert "strides" in _lib.last_error()
    for call, at in ((_packed, 2), (_paged, 3)):
        strides = [64] * (8 if call is _packed else 10)
        strides[at] = (1 << 25) + 8  # of K's tokens
        assert call(lib, strides=_lib.int64_array(strides)) == _lib.DSA_EUNSUPPORTED
    for at in (2, 5):  # of K's and V's pages
        strides = [64] * 10
        strides[at] = 1 << 35
        assert _paged(lib, strides=_lib.int64_array(strides)) == _lib.DSA_EUNSUPPORTED
        assert "page stride" in _lib.last_error()


def test_attention_refuses_too_many_tiles(lib):
    # 2^23 rows of 300 heads of their own: 2^16 tiles each, 19,660,800 of them.
    assert _packed(lib, q_rows=1 << 23, requests=1, heads=300, kv_heads=300,
                   workspace_bytes=1 << 60) == _lib.DSA_EUNSUPPORTED
    assert "tiles" in _lib.last_error()


@pytest.mark.parametrize("name,value,text", [
    ("page_size", 8, "page_size"), ("page_size", 24, "page_size"), ("page_size", -16, "page_size"),
    ("pages", -1, "page count"), ("table_stride", 3, "table"), ("table", None, "block table"),
    ("kv_lens", None, "lengths"), ("k_cache", None, "null"), ("table_width", -1, "table"),
])
def test_paged_attention_refusals(lib, name, value, text):
    assert _paged(lib, **{name: value}) < 0
    assert text in _lib.last_error()


def test_no_rows_is_no_call(lib):
    assert _packed(lib, q_rows=0, workspace=None, workspace_bytes=0) == _lib.DSA_OK
    assert _paged(lib, q_rows=0, workspace=None, workspace_bytes=0) == _lib.DSA_OK


def _plan(lib, **change):
    args = dict(cached=FAKE, fresh=FAKE, requests=2, table=FAKE, table_stride=4, table_width=4,
                free_pages=FAKE, free_count=3, page_size=16, tokens=8, q_start=FAKE, kv_lens=FAKE,
                slots=FAKE, status=FAKE, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_paged_plan(*args.values())


@pytest.mark.parametrize("name,value,text,status", [
    ("requests", -1, "negative", _lib.DSA_EINVAL),
    ("tokens", -1, "negative", _lib.DSA_EINVAL),
    ("free_count", -1, "negative", _lib.DSA_EINVAL),
    ("table_stride", 3, "overlap", _lib.DSA_EINVAL),
    ("page_size", 48, "page_size", _lib.DSA_EUNSUPPORTED),
    ("page_size", 0, "page_size", _lib.DSA_EUNSUPPORTED),
    ("requests", 8193, "8192", _lib.DSA_EUNSUPPORTED),
    *[(name, None, "null", _lib.DSA_EINVAL) for name in (
        "cached", "fresh", "table", "free_pages", "q_start", "kv_lens", "slots", "status")],
])
def test_plan_refusals(lib, name, value, text, status):
    assert _plan(lib, **{name: value}) == status
    assert text in _lib.last_error()


def _write(lib, **change):
    args = dict(k=FAKE, v=FAKE, k_cache=FAKE, v_cache=FAKE, strides=_lib.int64_array([256] * 10),
                tokens=4, heads=2, row_bytes=128, pages=3, page_size=16, slots=FAKE, stream=None)
    assert set(change) <= set(args)
    args.update(change)
    return lib.dsa_paged_write(*args.values())


@pytest.mark.parametrize("name,value,status", [
    ("tokens", -1, _lib.DSA_EINVAL), ("heads", 0, _lib.DSA_EINVAL),
    ("row_bytes", 0, _lib.DSA_EINVAL), ("pages", -1, _lib.DSA_EINVAL),
    ("strides", None, _lib.DSA_EINVAL), ("page_size", 17, _lib.DSA_EUNSUPPORTED),
    ("row_bytes", 40, _lib.DSA_EUNSUPPORTED), ("heads", 1 << 20, _lib.DSA_EUNSUPPORTED),
    ("strides", _lib.int64_array([256] * 9 + [24]), _lib.DSA_EINVAL),
    ("strides", _lib.int64_array([-256] + [256] * 9), _lib.DSA_EINVAL),
    ("k_cache", ctypes.c_void_p(4104), _lib.DSA_EINVAL),
    *[(name, None, _lib.DSA_EINVAL) for name in ("k", "v", "k_cache", "v_cache", "slots")],
])
def test_write_refusals(lib, name, value, status):
    assert _write(lib, **{name: value}) == status
    assert "dsa_paged_write" in _lib.last_error()


def test_nothing_to_write_is_no_call(lib):
    assert _write(lib, tokens=0) == _lib.DSA_OK
    assert _write(lib, pages=0) == _lib.DSA_OK


def test_workspace_sizes(lib):
    """Lists and partials by the host's bounds: q_rows G / tile rows + requests
    tiles, twice the chip's workgroups (512 of 128 rows, 256 of 16) of partials
    over all key heads where the keys may be cut, none where they are too few."""
    size = lib.dsa_seq_attention_workspace_bytes

    def expected(rows, requests, heads, kv, dim, keys):
        group = heads // kv
        narrow = rows * group <= 16 * requests
        tile, slots, uncut = (16, 256, 1024) if narrow else (128, 512, 640)
        tiles = max(1, rows * group // tile + requests)
        cut = keys > uncut and slots >= kv
        partials = 2 * slots // kv if cut else 0
        splits = min(tiles, partials // 2)
        at = 256 + 1024 + ((requests + 1) * 4 + 255) // 256 * 256 + (tiles + partials) * 64
        at += (splits * 64 + 255) // 256 * 256
        return at + partials * kv * tile * ((64 if dim <= 64 else 128) + 2) * 4

    for case in ((8, 2, 4, 2, 64, 100), (4, 4, 32, 8, 128, 1536), (64, 64, 64, 8, 128, 16384),
                 (2500, 8, 32, 8, 128, 30000), (32760, 1, 40, 8, 128, 32760), (3, 1, 3, 3, 40, 1024),
                 (3, 1, 3, 3, 40, 1025), (30, 1, 3, 3, 40, 640), (30, 1, 3, 3, 40, 641), (300, 2, 600, 600, 64, 10 ** 6), (5, 0, 1, 1, 8, 0)):
        assert size(*case) == expected(*case), case
    assert size(0, 3, 4, 2, 64, 100) == 0
    assert size(4, 3, 5, 2, 64, 100) == 0


def test_cpu_tensors_are_rejected():
    q, ints = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.packed_attention(q, q, q, ints)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q, cache, cache, torch.zeros((2, 4), dtype=torch.int32), ints[:2], ints)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_write(q, q, cache, cache, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_plan(ints, ints, torch.zeros((3, 4), dtype=torch.int32), ints, 16, 4)
