"""Attention scales without a GPU: those whose product with log2(e) leaves fp32 are
refused before any HIP call."""

import ctypes

import pytest

from dit_sparse_atten_amd import _lib

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


@pytest.mark.parametrize("scale", [2.36e38, 2.9e38, 3.4e38])
@pytest.mark.parametrize("paged", [False, True])
def test_scales_past_the_base_2_range(scale, paged):
    if not _lib.LIBRARY_PATH.exists():
        pytest.skip("libdsa.so not built")
    lib = _lib.load()
    tail = (scale, 1, 1, None, FAKE, 1 << 30, None)
    if paged:
        status = lib.dsa_paged_attention(FAKE, FAKE, FAKE, FAKE, 0, _lib.int64_array([64] * 10), 8,
                                         2, 4, 2, 64, 5, 16, FAKE, 4, 4, FAKE, FAKE, *tail)
    else:
        status = lib.dsa_packed_attention(FAKE, FAKE, FAKE, FAKE, 0, _lib.int64_array([64] * 8), 8,
                                          8, 2, 4, 2, 64, FAKE, None, *tail)
    assert status == _lib.DSA_EINVAL
    assert "scale" in _lib.last_error()
