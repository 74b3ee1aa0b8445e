"""The key/value cache's sizes and refusals: host code, no GPU."""
import ctypes as C

import numpy as np
import pytest

import kv_oracle as O
from tpu_compiler_amd import capi


def size(pages, page_tokens, heads, dim, bits):
    lib = capi.bind()
    return lib.tpuhip_kv_cache_bytes(C.byref(capi.KVDesc(pages, page_tokens, heads, dim, bits)))


@pytest.mark.parametrize("dim,padded", [(1, 64), (64, 64), (65, 96), (96, 96), (97, 128), (128, 128), (130, 192), (192, 192), (193, 256), (256, 256)])
@pytest.mark.parametrize("bits", [4, 8])
def test_bytes_of_a_cache(dim, padded, bits):
    assert size(3, 64, 5, dim, bits) == 3 * 64 * 5 * 2 * (padded * bits // 8 + 4)


def test_sizes_beyond_32_bits():
    assert size(1 << 20, 128, 8, 128, 4) == (1 << 27) * 8 * 136


@pytest.mark.parametrize("desc", [(0, 64, 1, 64, 4), (4, 63, 1, 64, 4), (4, 0, 1, 64, 4), (4, 64, 0, 64, 4), (4, 64, 65536, 64, 4),
                                  (4, 64, 1, 0, 4), (4, 64, 1, 257, 4), (4, 64, 1, 64, 3), (1 << 26, 32, 1, 64, 4), (-1, 64, 1, 64, 8)])
def test_sizes_that_are_refused(desc):
    assert size(*desc) == 0
    assert capi.bind().tpuhip_last_error()


def test_no_context_or_descriptor_is_refused():
    lib = capi.bind()
    assert lib.tpuhip_kv_cache_bytes(None) == 0
    assert lib.tpuhip_kv_cache_create(None, C.byref(capi.KVDesc(4, 64, 1, 64, 4)), C.byref(C.c_void_p())) == 1
    assert lib.tpuhip_kv_cache_destroy(None, None) == 1
    assert lib.tpuhip_kv_write(None, None, None, None) == 1 and lib.tpuhip_kv_read(None, None, None, None) == 1
    assert lib.tpuhip_kv_attention(None, None, None, None, None, None, None, None) == 1


@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
def test_the_oracle_by_heads_is_the_oracle(window, sinks):
    rng = np.random.default_rng(1)
    q = rng.standard_normal((12, 6, 8))
    k, v = ([rng.standard_normal((n, 2, 8)) for n in (20, 0, 3)] for _ in "kv")
    for a, b in zip(O.attention(q, k, v, [5, 2, 5], [20, 0, 3], 0.3, window, sinks), O.attention_of_finite(q, k, v, [5, 2, 5], [20, 0, 3], 0.3, window, sinks)):
        assert np.abs(a - b).max() < 1e-14
