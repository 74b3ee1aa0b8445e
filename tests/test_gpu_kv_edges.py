"""Attention to the key/value cache where numbers are far apart, and lengths and calls at their ends."""
import numpy as np
import pytest

import kv_bounds
import kv_oracle as O
from test_gpu_kv_cache import Sequences, ctx, rows  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def check(ctx, rng, q, q_lens, k, v, kv_lens, bits, dtype, page=32, **how):
    s = Sequences(ctx, rng, kv_lens, k[0].shape[1], k[0].shape[2], bits, page, k=k, v=v)
    got = s.attend(q, q_lens, dtype, **how)
    s.cache.close()
    want, limit = kv_bounds.attention(q, k, v, bits, q_lens, kv_lens, q.shape[2] ** -0.5, dtype, **how)
    off = np.abs(got - want) / limit
    assert off.max() <= 1, "%.3g of the bound at %s" % (off.max(), np.unravel_index(off.argmax(), off.shape))   # a NaN fails
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("first", ["zeros", "one number", "tiny"])
@pytest.mark.parametrize("size", [1e10, 1e25])
@pytest.mark.parametrize("q_len,heads,kv_heads,dim", [(1, 4, 2, 64), (9, 6, 2, 128), (70, 2, 2, 96), (60, 4, 2, 160)])
def test_values_that_grow_from_nothing(ctx, bits, first, size, q_len, heads, kv_heads, dim):
    """units whose values have a step of zero, or next to it, before values whose step is 2^29 and more"""
    rng = np.random.default_rng(1)
    n = 700
    k, v = (rows(rng, n, kv_heads, dim, "bf16", False) for _ in "kv")
    v[:600] = {"zeros": 0.0, "one number": 3.0, "tiny": O.rounded(v[:600] * 1e-35, "bf16")}[first]
    v[600:] = O.rounded(v[600:] * size, "bf16")
    q = rows(rng, q_len, heads, dim, "bf16", False)
    check(ctx, rng, q, [q_len], [k], [v], [n], bits, "bf16")
