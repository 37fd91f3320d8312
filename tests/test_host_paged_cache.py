"""The paged cache's C entry points without a GPU: refusals that come before any HIP
call."""

import ctypes

import pytest

from dit_sparse_atten_amd import _lib


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIBRARY_PATH.exists():
        pytest.skip("libdsa.so not built")
    return _lib.load()


FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


@pytest.mark.parametrize("tokens,heads,row_bytes", [
    (1 << 24, 128, 4080),            # a workgroup for each token
    ((1 << 28) + 16, 8, 256),        # 16 tokens for each
    (2 ** 31 - 1, 1, 32 * 1024),
    (2 ** 31 - 1, 12, 256),
])
def test_write_of_too_many_tokens(lib, tokens, heads, row_bytes):
    """More workgroups than a launch counts (K and V may be expanded, so that memory
    does not bound the tokens)."""
    status = lib.dsa_paged_write(FAKE, FAKE, FAKE, FAKE, _lib.int64_array([256] * 10), tokens,
                                 heads, row_bytes, 3, 16, FAKE, None)
    assert status == _lib.DSA_EUNSUPPORTED
    assert f"{tokens} tokens" in _lib.last_error()


@pytest.mark.parametrize("name", ["cached", "fresh", "table", "free_pages", "q_start", "kv_lens",
                                  "slots", "status"])
def test_plan_from_refusals(lib, name):
    args = dict(cached=FAKE, fresh=FAKE, requests=2, table=FAKE, table_stride=4, table_width=4,
                free_pages=FAKE, free_count=3, free_start=FAKE, page_size=16, tokens=8,
                q_start=FAKE, kv_lens=FAKE, slots=FAKE, status=FAKE, stream=None)
    args[name] = None
    assert lib.dsa_paged_plan_from(*args.values()) == _lib.DSA_EINVAL
    assert "null" in _lib.last_error()
