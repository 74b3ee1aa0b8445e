"""The key/value cache in 4 and 8 bits against its formulas in 64 bits."""
import numpy as np
import pytest

import gpu_capture
import kv_oracle as O
from tpu_compiler_amd import capi
from tpu_compiler_amd.kv_cache import DeviceArray, KVCache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context()
    yield c
    c.close()


def array(ctx, values, dtype):
    return DeviceArray.of(ctx, values, dtype)


class Strided:
    """rows of a part of a larger array"""

    def __init__(self, base, shape, stride, first):
        self.base, self.shape, self._stride, self.dtype = base, shape, stride, base.dtype
        self._ptr = base.data_ptr() + first * {"bf16": 2, "f16": 2, "f32": 4, "i32": 4}[base.dtype]

    def data_ptr(self):
        return self._ptr

    def stride(self):
        return self._stride


def rows(rng, n, heads, dim, dtype, spread=True):
    x = rng.standard_normal((n, heads, dim)) * rng.uniform(0.3, 2, (heads, dim)) + (rng.random((heads, dim)) < 0.1) * 4
    if spread:
        x *= 10.0 ** rng.integers(-2, 3, (n, heads, 1))
    return O.rounded(x, dtype)


def write_and_read(ctx, x, y, slots, bits, dtype, pages=8, page=64, read_slots=None):
    n, heads, dim = x.shape
    cache = KVCache(ctx, pages, heads, dim, bits, page)
    a = [array(ctx, v, dtype) for v in (x, y)]
    cache.write(*a, array(ctx, slots, "i32"))
    read_slots = slots if read_slots is None else read_slots
    out = [DeviceArray.of(ctx, np.full((len(read_slots), heads, dim), 7.0, np.float32), dtype) for _ in range(2)]
    cache.read(array(ctx, read_slots, "i32"), *out)
    got = [v.numpy().astype(np.float32) for v in out]
    cache.close()
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [1, 5, 63, 64, 65, 80, 96, 100, 128, 160, 192, 255, 256])
def test_rows_come_back_as_their_formula_says(ctx, bits, dtype, dim):
    """16-bit inputs: differences and quotients near a tie are far enough apart for 32 bits, every number is that of 64 bits"""
    rng = np.random.default_rng(dim * 10 + bits)
    n, heads = 70, 3
    x, y = rows(rng, n, heads, dim, dtype), rows(rng, n, heads, dim, dtype)
    for slots in (np.arange(n) + 64, np.arange(n) + 37, rng.permutation(512)[:n]):   # in order, not from a unit's start, anyhow
        for got, want in zip(write_and_read(ctx, x, y, slots, bits, dtype), (x, y)):
            assert np.array_equal(got, O.rounded(O.values(want, bits), dtype))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [33, 128])
def test_float32_rows_come_back_within_half_a_step(ctx, bits, dim):
    """32-bit inputs: x - m and its quotient are rounded, 2^-24 of at most 255 steps each, so that an element is at most
    (1/2 + 255 * 2^-22) steps off"""
    rng = np.random.default_rng(dim + bits)
    x, y = rows(rng, 100, 2, dim, "f32"), rows(rng, 100, 2, dim, "f32")
    for got, want in zip(write_and_read(ctx, x, y, np.arange(100) + 5, bits, "f32"), (x, y)):
        c, s, m = O.quantise(want, bits)
        # the step is a bfloat16: 32 bits round its quotient to the next one at most in one row of 2^15
        assert (np.abs(got - want.astype(np.float64)) <= s * (0.5 + 255 * 2.0 ** -22) * (1 + 2.0 ** -7)).all()
        assert (np.abs(got - (m + s * c)) <= 1e-6 * (np.abs(m) + s)).mean() > 0.999


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_of_special_numbers(ctx, bits):
    dim = 64
    r = np.random.default_rng(1).standard_normal(dim)
    special = [np.zeros(dim), -np.zeros(dim), np.full(dim, 3.0), np.full(dim, -1e-3), r * 1e37, r * 1e-37, r * 1e-39, r * 1e-42, r * 1e30,
               -np.abs(r) - 1, np.abs(r) + 1000, np.where(np.arange(dim) == 9, np.inf, r), np.where(np.arange(dim) == 60, -np.inf, r),
               np.where(np.arange(dim) == 0, np.nan, r), np.full(dim, np.nan), np.where(np.arange(dim) % 2, 3e38, -3e38),
               np.arange(dim) % 16, np.arange(dim) - 20.0, np.where(np.arange(dim) == 3, 1e38, 1.0)]
    x = O.rounded(np.array(special)[:, None], "bf16")
    for got in write_and_read(ctx, x, x[::-1].copy(), np.arange(len(x)) + 64, bits, "bf16"):
        want = O.rounded(O.values(x, bits), "bf16")
        assert np.isnan(want).all(-1).sum() == 5
        assert np.array_equal(got, want, equal_nan=True)
        x = x[::-1].copy()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,dim", [("bf16", 96), ("f32", 64), ("f16", 77)])
def test_parts_of_larger_arrays(ctx, bits, dtype, dim):
    """keys and values beside the queries in one array, out into another order of the axes"""
    rng = np.random.default_rng(3)
    n, heads = 45, 3
    qkv = rows(rng, n, 5 * heads + 1, dim, dtype, spread=False)
    base = array(ctx, qkv, dtype)
    stride = (base.shape[1] * dim, dim, 1)
    k, v = (Strided(base, (n, heads, dim), stride, i * heads * dim) for i in (2, 4))
    cache = KVCache(ctx, 4, heads, dim, bits, 32)
    slots = array(ctx, np.arange(n) + 11, "i32")
    cache.write(k, v, slots)
    for mark in (7.0,):
        out = array(ctx, np.full((2, heads, n + 1, dim + 2), mark, np.float32), dtype)
        ko, vo = (Strided(out, (n, heads, dim), (dim + 2, (n + 1) * (dim + 2), 1), i * heads * (n + 1) * (dim + 2) + 1) for i in range(2))
        cache.read(slots, ko, vo)
        got = out.numpy().astype(np.float32)
        for i, first in enumerate((2 * heads, 4 * heads)):
            want = O.rounded(O.values(qkv[:, first:first + heads], bits), dtype)
            if dtype != "f32":
                assert np.array_equal(got[i, :, :n, 1:-1], want.transpose(1, 0, 2))
            else:
                assert np.abs(got[i, :, :n, 1:-1] - want.transpose(1, 0, 2)).max() < 1
        untouched = np.ones_like(got, bool)
        untouched[:, :, :n, 1:-1] = False
        assert (got[untouched] == mark).all()
    cache.close()


@pytest.mark.parametrize("bits", [4, 8])
def test_writing_leaves_other_tokens_alone(ctx, bits):
    rng = np.random.default_rng(5)
    heads, dim, total = 2, 80, 192
    cache = KVCache(ctx, total // 32, heads, dim, bits, 32)
    every = array(ctx, np.arange(total), "i32")
    out = [DeviceArray(ctx, (total, heads, dim), "bf16") for _ in range(2)]
    held = np.zeros((2, total, heads, dim), np.float32)
    cache.read(every, *out)
    assert all(np.array_equal(o.numpy(), held[0]) for o in out)          # fresh pages
    for slots in (np.arange(total), [3], [31, 32, 33, 34, 35], np.arange(60, 101), [4, 5, 6, 7, 191, 0, 2, 1, 3], np.arange(64, 96),
                  [-1, 17, total, 2 ** 31 - 1, -2 ** 31, 18, 19], np.arange(40)[::-1]):
        slots = np.asarray(slots)
        x, y = rows(rng, len(slots), heads, dim, "bf16"), rows(rng, len(slots), heads, dim, "bf16")
        cache.write(array(ctx, x, "bf16"), array(ctx, y, "bf16"), array(ctx, slots, "i32"))
        there = (slots >= 0) & (slots < total)
        held[0, slots[there]], held[1, slots[there]] = x[there], y[there]
        cache.read(every, *out)
        for o, h in zip(out, held):
            assert np.array_equal(o.numpy(), O.rounded(O.values(h, bits), "bf16"))
    got = DeviceArray.of(ctx, np.full((3, heads, dim), 7.0), "f32"), DeviceArray.of(ctx, np.full((3, heads, dim), 7.0), "f32")
    cache.read(array(ctx, [-1, 2, total], "i32"), *got)
    for o, h in zip(got, held):
        assert not o.numpy()[[0, 2]].any() and np.array_equal(o.numpy()[1], O.values(h[2], bits))
    cache.close()


class Sequences:
    """sequences in a cache, their pages in an order of no meaning, and what 64 bits hold of them"""

    def __init__(self, ctx, rng, kv_lens, heads, dim, bits, page=64, dtype="bf16", k=None, v=None, spare=3, first_page=0):
        self.ctx, self.kv_lens, self.page = ctx, list(kv_lens), page
        need = [-(-n // page) for n in kv_lens]
        self.cache = KVCache(ctx, first_page + sum(need) + spare, heads, dim, bits, page)
        order = first_page + rng.permutation(sum(need) + spare)
        self.table = np.full((len(need), max(need + [1])), -1, np.int64)
        self.k, self.v, at = [], [], 0
        for i, n in enumerate(kv_lens):
            self.table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
            kk = rows(rng, n, heads, dim, dtype, spread=False) if k is None else k[i]
            vv = rows(rng, n, heads, dim, dtype, spread=False) if v is None else v[i]
            slots = self.table[i][np.arange(n) // page] * page + np.arange(n) % page
            if n:
                self.cache.write(array(ctx, kk, dtype), array(ctx, vv, dtype), array(ctx, slots, "i32"))
            self.k.append(O.values(kk, bits) if n else kk.astype(np.float64))
            self.v.append(O.values(vv, bits) if n else vv.astype(np.float64))

    def attend(self, q, q_lens, dtype, table=None, out=None, **how):
        a, ctx = array(self.ctx, q, dtype), self.ctx
        o = DeviceArray.of(ctx, np.full(q.shape, 7.0, np.float32), dtype) if out is None else out
        self.cache.attention(a, o, array(ctx, np.cumsum([0] + list(q_lens)), "i32"), array(ctx, self.kv_lens, "i32"),
                             array(ctx, self.table if table is None else table, "i32"), **how)
        return o.numpy().astype(np.float64)


def bound(q, seqs, want, size, scale, dtype, least=2.0 ** -24):
    """How far a result may be: its own rounding (half a unit of 8 or 11 bits), a weight's rounding to float16 (2^-11 of every
    term of the sum; the other half for the weights of the sum they are divided by), and the scores' sums in 32 bits: at most 300
    roundings of terms that come to T, which weights feel in full, twice."""
    def terms(x):     # m and s c apart are at most three times the largest |value|
        return max([np.abs(np.where(np.isfinite(v), v, 0)).max() for v in x if v.size] + [0.0])
    t = 3 * np.abs(q).sum(-1, keepdims=True) * terms(seqs.k) * scale
    unit = {"bf16": 2.0 ** -9, "f16": 2.0 ** -11}[dtype]
    offsets = terms(seqs.v)        # the sum of offsets and the sum of codes may cancel
    return unit * np.abs(want) + (2.0 ** -10 + 2 * 300 * 2.0 ** -24 * t) * (size + 3 * offsets) + least


def check(rng, ctx, kv_lens, q_lens, heads, kv_heads, dim, bits, dtype, page=64, scale=None, q=None, k=None, v=None, oracle=O.attention, **how):
    s = Sequences(ctx, rng, kv_lens, kv_heads, dim, bits, page, k=k, v=v)
    if q is None:
        q = rows(rng, sum(q_lens), heads, dim, dtype, spread=False)
    used = dim ** -0.5 if scale is None else scale
    want, size = oracle(q, s.k, s.v, q_lens, kv_lens, used, **how)
    got = s.attend(q, q_lens, dtype, scale=scale, **how)
    limit = bound(q, s, want, size, used, dtype)
    s.cache.close()
    assert np.isfinite(got).all()
    off = np.abs(got - want) / limit
    assert off.max(initial=0) <= 1, "%.3g of the bound at %s" % (off.max(), np.unravel_index(off.argmax(), off.shape))
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kv", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 700])
def test_single_tokens(ctx, bits, kv):
    check(np.random.default_rng(kv), ctx, [kv], [1], 8, 2, 128, bits, "bf16")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (12, 4), (7, 1), (16, 1), (17, 1), (40, 2), (64, 1), (65, 1), (130, 1)])
def test_shared_heads(ctx, heads, kv_heads):
    rng = np.random.default_rng(heads)
    check(rng, ctx, [150], [1], heads, kv_heads, 64, 4, "bf16")
    check(rng, ctx, [90, 41], [3, 5], heads, kv_heads, 64, 4, "f16")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [1, 7, 32, 64, 72, 80, 96, 112, 128, 144, 192, 200, 256])
def test_head_sizes(ctx, bits, dim):
    rng = np.random.default_rng(dim)
    check(rng, ctx, [100, 37], [1, 1], 4, 2, dim, bits, "bf16")
    check(rng, ctx, [100, 37], [30, 9], 6, 2, dim, bits, "f16", page=32)
    check(rng, ctx, [300], [270], 2, 2, dim, bits, "bf16")


@pytest.mark.parametrize("bits,dtype", [(4, "bf16"), (8, "f16")])
@pytest.mark.parametrize("q,kv", [(2, 2), (5, 64), (17, 40), (33, 33), (64, 500), (65, 65), (129, 400), (300, 300)])
def test_prompts_and_parts_of_them(ctx, bits, dtype, q, kv):
    check(np.random.default_rng(q), ctx, [kv, kv + 9], [q, max(1, q - 1)], 4, 2, 128, bits, dtype)


@pytest.mark.parametrize("bits,dim,dtype", [(4, 64, "bf16"), (8, 80, "f16"), (4, 128, "f16"), (8, 128, "bf16"), (4, 200, "bf16"), (8, 250, "f16")])
@pytest.mark.parametrize("q,kv,heads,kv_heads", [(41, 250, 96, 3), (150, 230, 70, 7), (270, 290, 50, 2), (270, 290, 96, 8), (270, 290, 260, 4), (60, 1500, 12, 1)])
def test_many_rows(ctx, bits, dim, dtype, q, kv, heads, kv_heads):
    """so many that each form of the kernel has its turn: 16 to 128 rows a workgroup, of which one to four waves have their own"""
    rng = np.random.default_rng(q + heads)
    check(rng, ctx, [kv, 40], [q, 7], heads, kv_heads, dim, bits, dtype, page=32, oracle=O.attention_of_finite)
    check(rng, ctx, [kv], [q], heads, kv_heads, dim, bits, dtype, window=kv // 3, sinks=33, oracle=O.attention_of_finite)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (32, 0), (33, 4), (64, 40), (100, 64), (1000, 3), (7, 1000)])
def test_windows_and_first_tokens(ctx, window, sinks):
    rng = np.random.default_rng(window)
    check(rng, ctx, [1, 40, 333, 610], [1, 1, 1, 1], 4, 2, 64, 4, "bf16", window=window, sinks=sinks)
    check(rng, ctx, [333, 150], [70, 150], 4, 2, 64, 4, "f16", window=window, sinks=sinks, page=32)
    check(rng, ctx, [800], [3], 6, 1, 128, 8, "bf16", window=window, sinks=sinks, page=128)


def test_many_tokens_of_one_and_of_several_sequences(ctx):
    rng = np.random.default_rng(0)
    check(rng, ctx, [9000], [1], 8, 1, 64, 4, "bf16")
    check(rng, ctx, [5000, 1, 2345, 64], [2, 1, 3, 1], 4, 2, 128, 4, "f16")
    check(rng, ctx, [6000], [1], 4, 2, 64, 4, "bf16", window=4000, sinks=5)
    check(rng, ctx, [4100], [40], 4, 1, 96, 8, "bf16")


def test_lengths_of_nothing(ctx):
    """no tokens, no queries, more queries than tokens: zeros where nothing is to be seen"""
    rng = np.random.default_rng(2)
    got = check(rng, ctx, [0, 5, 70, 3], [2, 0, 1, 6], 4, 2, 64, 4, "bf16")
    assert not got[:2].any() and not got[3:6].any() and got[6:].any()
    s = Sequences(ctx, rng, [10], 2, 64, 4)
    assert s.attend(np.zeros((0, 4, 64), np.float32), [0], "bf16").size == 0
    s.cache.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_sizes_of_queries_keys_and_values(ctx, dtype):
    """large and small numbers, one key above all others, rows of one number"""
    rng = np.random.default_rng(4)
    n, d = 200, 64
    k, v = rows(rng, n, 2, d, "bf16", False), rows(rng, n, 2, d, "bf16", False)
    q = rows(rng, 3, 4, d, dtype, False)
    for a, b, c in ((100, 1, 1), (1e-4, 1, 1), (1, 1e-6, 1), (0.01, 300, 1)):
        check(rng, ctx, [n], [3], 4, 2, d, 4, dtype, q=O.rounded(q * a, dtype), k=[O.rounded(k * b, "bf16")], v=[O.rounded(v * c, "bf16")])
    high = k.copy()
    high[77] *= 30
    check(rng, ctx, [n], [3], 4, 2, d, 4, dtype, q=q, k=[O.rounded(high, "bf16")], v=[v])
    check(rng, ctx, [n], [3], 4, 2, d, 8, dtype, q=q, k=[np.ones_like(k)], v=[v])
    check(rng, ctx, [n], [3], 4, 2, d, 8, dtype, q=np.zeros_like(q), k=[k], v=[np.full_like(v, -2.5)])
    check(rng, ctx, [n], [3], 4, 2, d, 4, dtype, q=q, k=[k], v=[v], scale=0.0)
    check(rng, ctx, [n], [3], 4, 2, d, 4, dtype, q=q, k=[k], v=[v], scale=-0.3)


@pytest.mark.parametrize("size", [1e-30, 1e-8, 1e8, 1e30])
def test_values_of_any_size(ctx, size):
    """steps of the values far from one, and of every size in one cache: relative to the largest"""
    rng = np.random.default_rng(6)
    n, d = 300, 64
    k, v = rows(rng, n, 1, d, "bf16", False), rows(rng, n, 1, d, "bf16", False)
    for change in (np.full((n, 1, 1), size), size ** rng.random((n, 1, 1)), size ** (np.arange(n) / n)[:, None, None]):
        s = Sequences(ctx, rng, [n], 1, d, 4, k=[k], v=[O.rounded(v * change, "bf16")])
        q = rows(rng, 2, 4, d, "bf16", False)
        want, total = O.attention(q, s.k, s.v, [2], [n], 0.125)
        got = s.attend(q, [2], "bf16")
        limit = bound(q, s, want, total, 0.125, "bf16", least=0)
        assert (np.abs(got - want) <= limit).all()
        s.cache.close()


def test_what_is_masked_does_not_count(ctx):
    """rows that hold NaN, in places that some queries see and others do not, and pages that are no longer there"""
    rng = np.random.default_rng(7)
    n, d = 260, 64
    for q_len, window, sinks in ((1, 50, 4), (40, 50, 4), (200, 30, 2), (7, 64, 0)):
        k, v = rows(rng, n, 2, d, "bf16", False), rows(rng, n, 2, d, "bf16", False)
        first = n - q_len                            # the first query's position
        for x, hidden in ((k, first - window - 10), (v, first - window - 3), (v, n - 1)):
            if hidden >= sinks:
                x[hidden] = np.nan
        s = Sequences(ctx, rng, [n], 2, d, 4, page=32, k=[k], v=[v])
        q = rows(rng, q_len, 4, d, "bf16", False)
        want, size = O.attention(q, s.k, s.v, [q_len], [n], 0.125, window, sinks)
        table = s.table.copy()
        table[0, -(-sinks // 32):max(-(-sinks // 32), (first - window + 1) // 32)] = -5
        table[0, 1] = table[0, 1] if table[0, 1] >= 0 else 2 ** 31 - 1
        got = s.attend(q, [q_len], "bf16", table=table, window=window, sinks=sinks)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.isnan(want[-1]).all()
        fine = ~np.isnan(want)
        if q_len > 1:
            assert fine[:-1].all()
        limit = bound(q, s, np.where(fine, want, 0), np.where(fine, size, 0), 0.125, "bf16")
        assert (np.abs(got - want)[fine] <= limit[fine]).all()
        s.cache.close()


def test_a_query_that_is_not_finite_harms_itself_alone(ctx):
    rng = np.random.default_rng(8)
    s = Sequences(ctx, rng, [90], 1, 64, 4)
    q = rows(rng, 5, 2, 64, "bf16", False)
    want, size = O.attention(q, s.k, s.v, [5], [90], 0.125)
    q[2, 1, 7], q[4, 0, 0] = np.inf, np.nan
    got = s.attend(q, [5], "bf16")
    harmed = np.zeros((5, 2), bool)
    harmed[2, 1] = harmed[4, 0] = True
    assert np.isnan(got[harmed]).all()
    q[harmed] = 0
    assert (np.abs(got - want)[~harmed] <= bound(q, s, want, size, 0.125, "bf16")[~harmed]).all()
    s.cache.close()


def test_strides_of_queries_and_results(ctx):
    """heads before tokens, an odd distance of rows; what lies between the rows stays"""
    rng = np.random.default_rng(9)
    n, heads, d = 21, 6, 64
    for dim in (64, 61):
        s = Sequences(ctx, rng, [50], 2, dim, 4)
        wide = rows(rng, heads, n, d + 1, "bf16", False)
        base, out = array(ctx, wide, "bf16"), array(ctx, np.full((heads, n, d + 1), 7.0), "bf16")
        stride = (d + 1, n * (d + 1), 1)
        s.cache.attention(Strided(base, (n, heads, dim), stride, 1), Strided(out, (n, heads, dim), stride, 1), array(ctx, [0, n], "i32"),
                          array(ctx, [50], "i32"), array(ctx, s.table, "i32"))
        q = wide[:, :, 1:dim + 1].transpose(1, 0, 2)
        want, size = O.attention(q, s.k, s.v, [n], [50], dim ** -0.5)
        got = out.numpy().astype(np.float64)
        assert (np.abs(got[:, :, 1:dim + 1].transpose(1, 0, 2) - want) <= bound(q, s, want, size, dim ** -0.5, "bf16")).all()
        assert (got[:, :, 0] == 7).all() and (got[:, :, dim + 1:] == 7).all()
        s.cache.close()


def test_rows_between_sequences_and_beyond_the_bounds_stay(ctx):
    """what the lengths on the device say is cut to what the call says: more queries or tokens than that are not looked at"""
    rng = np.random.default_rng(10)
    s = Sequences(ctx, rng, [70, 90], 1, 64, 4)
    q = rows(rng, 12, 2, 64, "bf16", False)
    out = array(ctx, np.full((12, 2, 64), 7.0), "bf16")
    s.cache.attention(array(ctx, q, "bf16"), out, array(ctx, [-3, 4, 4000], "i32"), array(ctx, [70, 9000], "i32"), array(ctx, s.table, "i32"),
                      max_q=4, max_kv=90)
    got = out.numpy().astype(np.float64)
    want, size = O.attention(q[:8], s.k, s.v, [4, 4], [70, 90], 0.125)
    assert (np.abs(got[:8] - want) <= bound(q[:8], s, want, size, 0.125, "bf16")).all()
    assert (got[8:] == 7).all()
    s.cache.close()


def test_offsets_beyond_32_bits(ctx):
    """a cache of 5 GiB, a sequence at its end"""
    rng = np.random.default_rng(11)
    heads, dim, page = 8, 256, 128
    unit_page = 2 * page * (dim + 4) * heads
    first = 5 * 2 ** 30 // unit_page
    s = Sequences(ctx, rng, [300, 40], heads, dim, 8, page, first_page=first)
    assert s.cache.nbytes > 2 ** 32
    q = rows(rng, 2, 16, dim, "bf16", False)
    want, size = O.attention(q, s.k, s.v, [1, 1], [300, 40], dim ** -0.5)
    got = s.attend(q, [1, 1], "bf16")
    assert (np.abs(got - want) <= bound(q, s, want, size, dim ** -0.5, "bf16")).all()
    out = [DeviceArray(ctx, (40, heads, dim), "f32") for _ in range(2)]
    slots = s.table[1][0] * page + np.arange(40)
    s.cache.read(array(ctx, slots, "i32"), *out)
    assert np.array_equal(out[0].numpy(), s.k[1]) and np.array_equal(out[1].numpy(), s.v[1])
    s.cache.close()


def test_a_captured_step_replays(ctx):
    """one token written and attended to, recorded once; lengths, slots and rows are those of the moment it runs"""
    rng = np.random.default_rng(12)
    heads, d, page = 2, 64, 32
    s = Sequences(ctx, rng, [3000, 45], heads, d, 4, page)
    extra = [array(ctx, np.zeros((2, heads, d)), "bf16") for _ in range(2)]
    q, out = array(ctx, np.zeros((2, 4, d)), "bf16"), DeviceArray(ctx, (2, 4, d), "bf16")
    slots, lens = array(ctx, [-1, -1], "i32"), array(ctx, s.kv_lens, "i32")
    table = array(ctx, s.table, "i32")
    starts = array(ctx, [0, 1, 2], "i32")
    write = s.cache.plan_write(*extra, slots)
    attend = s.cache.plan_attention(q, out, starts, lens, table, max_q=1, max_kv=3008)
    write(), attend()                                # once before it is recorded
    graph = gpu_capture.Graph(ctx.h)
    with graph.recording():
        write()
        attend()
    for step in range(3):
        new, qs = rows(rng, 4, heads, d, "bf16", False).reshape(2, 2, heads, d), rows(rng, 2, 4, d, "bf16", False)
        at = []
        for i in range(2):
            n = s.kv_lens[i]
            at.append(s.table[i][n // page] * page + n % page)
            s.k[i] = np.concatenate([s.k[i], O.values(new[0, i:i + 1], 4)])
            s.v[i] = np.concatenate([s.v[i], O.values(new[1, i:i + 1], 4)])
            s.kv_lens[i] += 1
        as_bf16 = lambda x: (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
        for x, y in zip(extra, new):
            ctx.upload(x.ptr, as_bf16(y))
        ctx.upload(q.ptr, as_bf16(qs))
        ctx.upload(slots.ptr, np.array(at, np.int32))
        ctx.upload(lens.ptr, np.array(s.kv_lens, np.int32))
        graph.replay()
        got = out.numpy().astype(np.float64)
        want, size = O.attention(qs, s.k, s.v, [1, 1], s.kv_lens, 0.125)
        assert (np.abs(got - want) <= bound(qs, s, want, size, 0.125, "bf16")).all()
        attend()                                     # the same, not replayed
        assert np.array_equal(out.numpy(), got.astype(np.float32))
    graph.close()
    s.cache.close()


def test_another_context_and_repeated_calls(ctx):
    """a cache used from another context of its device; the same call gives the same bits"""
    rng = np.random.default_rng(13)
    s = Sequences(ctx, rng, [4000], 2, 128, 4)
    q = rows(rng, 1, 16, 128, "bf16", False)
    first = s.attend(q, [1], "bf16")
    for _ in range(5):
        assert np.array_equal(s.attend(q, [1], "bf16"), first)
    ctx.sync()
    other = capi.Context()
    out = DeviceArray(other, (1, 16, 128), "bf16")
    a = [array(other, x, t) for x, t in ((q, "bf16"), ([0, 1], "i32"), ([4000], "i32"), (s.table, "i32"))]
    d = capi.KVAttentionDesc(1, 16, 0, 1, 1, 4000, 0, 0, s.table.shape[1], 128 ** -0.5, 2048, 128, 2048, 128)
    capi.check(other.lib, other.lib.tpuhip_kv_attention(other.h, s.cache.h, d, a[0].ptr, out.ptr, a[1].ptr, a[2].ptr, a[3].ptr))
    assert np.array_equal(out.numpy().astype(np.float64), first)
    other.close()
    s.cache.close()


def test_a_context_on_the_stream_of_another(ctx):
    rng = np.random.default_rng(14)
    s = Sequences(ctx, rng, [100], 2, 64, 4)
    q = rows(rng, 1, 4, 64, "bf16", False)
    want = s.attend(q, [1], "bf16")
    other = capi.Context(stream=ctx.lib.tpuhip_ctx_stream(ctx.h))
    s.cache.ctx, s.ctx = other, other                # what the first one has issued is before this
    assert np.array_equal(s.attend(q, [1], "bf16"), want)
    s.cache.close()
    other.close()


def test_page_tables_whose_rows_end_early(ctx):
    """the last sequence's row of a table ends where its pages do, whatever the distance of rows"""
    rng = np.random.default_rng(15)
    s = Sequences(ctx, rng, [70, 130], 1, 64, 4, page=32)
    q = rows(rng, 2, 2, 64, "bf16", False)
    want = s.attend(q, [1, 1], "bf16")
    wide = np.full((2, 40), -1)
    wide[:, 40 - s.table.shape[1]:] = s.table
    base = array(ctx, wide, "i32")
    out = DeviceArray(ctx, q.shape, "bf16")
    s.cache.attention(array(ctx, q, "bf16"), out, array(ctx, [0, 1, 2], "i32"), array(ctx, [70, 130], "i32"),
                      Strided(base, s.table.shape, (40, 1), 40 - s.table.shape[1]))
    assert np.array_equal(out.numpy().astype(np.float64), want)
    s.cache.close()


def test_refusals(ctx):
    for sizes in ((0, 1, 64, 4, 64), (4, 0, 64, 4, 64), (4, 1, 0, 4, 64), (4, 1, 257, 4, 64), (4, 1, 64, 5, 64), (4, 1, 64, 4, 48),
                  (4, 1, 64, 4, 0), (1 << 26, 1, 64, 4, 32), (4, 70000, 64, 4, 32)):
        with pytest.raises(capi.TpuHipError):
            KVCache(ctx, *sizes)
    cache = KVCache(ctx, 4, 2, 64, 4, 32)
    x, y = DeviceArray(ctx, (5, 2, 64), "bf16"), DeviceArray(ctx, (5, 2, 64), "f16")
    slots = array(ctx, np.arange(5), "i32")
    refused = lambda f, *a, **k: pytest.raises(capi.TpuHipError, f, *a, **k)
    refused(cache.write, x, y, slots)
    refused(cache.write, x, x, array(ctx, np.arange(4), "i32"))
    refused(cache.write, x, x, DeviceArray(ctx, (5,), "f32"))
    refused(cache.write, DeviceArray(ctx, (5, 3, 64), "bf16"), x, slots)
    refused(cache.write, Strided(x, (5, 2, 64), (128, 64, 2), 0), x, slots)
    refused(cache.read, slots, Strided(x, (5, 2, 64), (64, 64, 1), 0), x)
    refused(cache.write, Strided(x, (5, 2, 64), (-128, 64, 1), 0), x, slots)
    q, starts, lens = DeviceArray(ctx, (3, 4, 64), "bf16"), array(ctx, [0, 3], "i32"), array(ctx, [3], "i32")
    table = array(ctx, [[0, 1]], "i32")
    cache.attention(q, DeviceArray(ctx, (3, 4, 64), "bf16"), starts, lens, table)
    for a in ((DeviceArray(ctx, (3, 5, 64), "bf16"),) * 2, (DeviceArray(ctx, (3, 4, 64), "f32"),) * 2, (q, y), (q, DeviceArray(ctx, (2, 4, 64), "bf16")),
              (q, Strided(q, (3, 4, 64), (64, 64, 1), 0))):
        refused(cache.attention, *a, starts, lens, table)
    refused(cache.attention, q, q, starts, lens, table)             # in place
    for how in (dict(max_kv=65), dict(window=-1), dict(sinks=-1), dict(scale=float("nan")), dict(max_q=-1), dict(max_kv=-1)):
        refused(cache.attention, q, q, starts, lens, table, **how)
    refused(cache.attention, q, q, starts, array(ctx, [3, 3], "i32"), table)
    refused(cache.attention, q, q, array(ctx, [0], "i32"), lens, table)
    lib = ctx.lib
    assert lib.tpuhip_kv_write(ctx.h, None, None, None) == 1 and lib.tpuhip_kv_attention(None, cache.h, None, *[None] * 5) == 1
    assert lib.tpuhip_kv_cache_create(ctx.h, None, None) == 1 and lib.tpuhip_kv_cache_bytes(None) == 0
    rows = capi.KVRows(3, 7, q.ptr, q.ptr, 128, 64, 128, 64)
    assert lib.tpuhip_kv_read(ctx.h, cache.h, rows, slots.ptr) == 1 and b"type" in lib.tpuhip_last_error()
    rows = capi.KVRows(3, 0, None, q.ptr, 128, 64, 128, 64)
    assert lib.tpuhip_kv_read(ctx.h, cache.h, rows, slots.ptr) == 1
    rows = capi.KVRows(2 ** 30, 0, q.ptr, q.ptr, 128, 64, 128, 64)
    assert lib.tpuhip_kv_write(ctx.h, cache.h, rows, slots.ptr) == 1 and b"one call" in lib.tpuhip_last_error()
    rows = capi.KVRows(0, 0, None, None, 0, 0, 0, 0)
    assert lib.tpuhip_kv_read(ctx.h, cache.h, rows, None) == 0      # nothing to do
    cache.close()
    cache.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_the_example_answers_as_with_exact_rows(ctx, window, sinks):
    """prompts of different lengths, then single tokens: the logits are those of attention in 64 bits to the rows that the cache holds
    of the same tokens.  Rows, queries and results are bfloat16 there and here, so that a step's logits differ by roundings of 2^-9 alone:
    of a layer's result (twice, of what it adds), and of numbers that these move to the next one (four times as many, in three
    layers); relative to logits of size one, 64 * 2^-9 is far above that and far below what a wrong token does."""
    from tpu_compiler_amd import kv_example
    model = kv_example.Model()
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 512, n) for n in (3, 130, 64, 1)]
    answers, steps, _ = kv_example.generate(ctx, model, prompts, 5, 8, window, sinks, page_tokens=32)
    for i, prompt in enumerate(prompts):
        held = [([], []) for _ in model.qkv]

        def attend(layer, q, k, v):
            for x, y in zip(held[layer], (k, v)):
                x.append(O.values(O.rounded(y, "bf16"), 8))
            kk, vv = (np.concatenate(x) for x in held[layer])
            return O.rounded(O.attention(O.rounded(q, "bf16"), [kk], [vv], [len(q)], [len(kk)], 0.125, window, sinks)[0], "bf16")

        new = prompt
        for step, answer in zip(steps, answers[i]):
            want = model(np.asarray(new), attend)[-1]
            assert np.abs(step[i] - want).max() <= 64 * 2.0 ** -9
            new = [answer]                           # the example's own, should two be alike
