"""Attention to the key/value cache where numbers are far apart, and lengths and calls at their ends."""
import os
import subprocess
import sys

import numpy as np
import pytest

import kv_bounds
import kv_oracle as O
from test_gpu_kv_cache import Sequences, Strided, array, ctx, rows  # noqa: F401 (a fixture)
from tpu_compiler_amd import capi
from tpu_compiler_amd.kv_cache import DeviceArray, KVCache

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


@pytest.mark.parametrize("dim", [64, 128, 200])
@pytest.mark.parametrize("q_len", [1, 20, 300])
def test_sequences_that_are_all_empty(ctx, dim, q_len):
    """no page and no token: zeros, by a table of no columns"""
    cache = KVCache(ctx, 2, 2, dim, 4, 32)
    q = array(ctx, np.ones((3 * q_len, 4, dim)), "bf16")
    out = array(ctx, np.full((3 * q_len, 4, dim), 7.0), "bf16")
    starts, lens = array(ctx, np.arange(4) * q_len, "i32"), array(ctx, np.zeros(3), "i32")
    cache.attention(q, out, starts, lens, DeviceArray(ctx, (3, 0), "i32"))
    assert not out.numpy().any()
    cache.attention(q, out, starts, lens, DeviceArray(ctx, (3, 2), "i32"), max_q=q_len, max_kv=0)
    assert not out.numpy().any()
    cache.close()


@pytest.mark.parametrize("size", [1e6, 1e10, 1e25])
@pytest.mark.parametrize("q_len,window,sinks", [(1, 40, 3), (1, 64, 0), (5, 40, 3), (70, 0, 0), (70, 33, 5)])
@pytest.mark.parametrize("bits,dim", [(4, 64), (8, 128), (4, 160)])
def test_large_values_where_a_query_does_not_look(ctx, bits, dim, size, q_len, window, sinks):
    """finite numbers in hidden places, beside tokens that are seen in one unit: before the window, behind the first tokens, later than the query"""
    rng = np.random.default_rng(2)
    n = 300
    k, v = (rows(rng, n, 2, dim, "bf16", False) for _ in "kv")
    first = n - q_len
    hidden = [t for t in (first - window - 1, first - window, sinks, sinks + 1) if window and sinks <= t <= first - window]
    hidden += [n - 1, n - 17] if q_len > 20 else []
    assert hidden
    v[hidden] = O.rounded(v[hidden] * size, "bf16")
    q = rows(rng, q_len, 4, dim, "bf16", False)
    check(ctx, rng, q, [q_len], [k], [v], [n], bits, "bf16", window=window, sinks=sinks)


@pytest.mark.parametrize("n,at", [(1, 0), (40, 39), (300, 3), (300, 150), (5000, 4999), (9000, 70)])
def test_scores_far_below_zero(ctx, n, at):
    """the largest of them is what the others are relative to, however low it is: one of -2.4e34 among others of -2.4e35, which is far more
    apart than the roundings of such numbers, has all the weight, and its values come back as they are held"""
    rng = np.random.default_rng(3)
    k, v = np.full((n, 1, 64), 3e17, np.float32), rows(rng, n, 1, 64, "bf16", False)
    k[at] = 3e16
    q = np.full((1, 2, 64), -1e17, np.float32)
    k, q = O.rounded(k, "bf16"), O.rounded(q, "bf16")
    s = Sequences(ctx, rng, [n], 1, 64, 4, 32, k=[k], v=[v])
    got = s.attend(q, [1], "bf16")
    s.cache.close()
    assert np.array_equal(got[0], np.repeat(O.rounded(O.values(v[at], 4), "bf16").astype(np.float64), 2, 0))


@pytest.mark.parametrize("n,at", [(70, 3), (70, 66), (64, 40), (300, 150)])
@pytest.mark.parametrize("q_len", [1, 20])
def test_a_row_that_cannot_be_held_shows_whatever_its_weight(ctx, n, at, q_len):
    """a query sees values that are NaN with a weight that 32 bits do not hold: not a number, in a unit that is seen as a whole or in part"""
    rng = np.random.default_rng(4)
    k, v = (rows(rng, n, 1, 64, "bf16", False) for _ in "kv")
    q = np.abs(rows(rng, q_len, 2, 64, "bf16", False))
    k[:], k[at] = 0, -100
    v[at] = np.nan
    s = Sequences(ctx, rng, [n], 1, 64, 4, 32, k=[k], v=[v])
    got = s.attend(q, [q_len], "bf16")
    s.cache.close()
    sees = n - q_len + np.arange(q_len) >= at
    assert np.isnan(got[sees]).all() and not np.isnan(got[~sees]).any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [40, 100, 20000])
def test_a_slot_twice_for_the_same_row(ctx, bits, n):
    """in one unit's run and outside of it, in one workgroup and in several"""
    rng = np.random.default_rng(5)
    cache = KVCache(ctx, -(-n // 32) + 1, 2, 80, bits, 32)
    x, y = rows(rng, n, 2, 80, "bf16", False), rows(rng, n, 2, 80, "bf16", False)
    which = np.concatenate([np.arange(n), rng.integers(0, n, n // 2), np.full(9, n // 3), [n - 1]])
    which = np.concatenate([which[:n // 2], which[n:], which[n // 2:n]])
    cache.write(array(ctx, x[which], "bf16"), array(ctx, y[which], "bf16"), array(ctx, which, "i32"))
    got = [DeviceArray(ctx, (n + 8, 2, 80), "bf16") for _ in range(2)]
    cache.read(array(ctx, np.arange(n + 8), "i32"), *got)
    for a, b in zip(got, (x, y)):
        held = a.numpy()
        assert np.array_equal(held[:n], O.rounded(O.values(b, bits), "bf16")) and not held[n:].any()
    cache.close()


def test_each_refusal_says_what_it_is(ctx):
    """one thing wrong at a time, beside a call that is taken"""
    cache = KVCache(ctx, 4, 2, 64, 4, 32)
    q, out = (DeviceArray(ctx, (3, 4, 64), "bf16") for _ in range(2))
    starts, lens, table = array(ctx, [0, 3], "i32"), array(ctx, [3], "i32"), array(ctx, [[0, 1]], "i32")
    good = dict(q=q, out=out, q_starts=starts, kv_lens=lens, page_table=table)
    other = lambda heads, dtype, n=3: DeviceArray(ctx, (n, heads, 64), dtype)
    cache.attention(**good)
    for change, says in ((dict(max_kv=65), "65 tokens in 2 pages"), (dict(max_kv=-1), "of -1 tokens"), (dict(max_q=-1), "at most -1 a sequence"),
                         (dict(window=-1), "window of -1"), (dict(sinks=-1), "-1 first tokens"), (dict(scale=float("nan")), "not finite"),
                         (dict(scale=float("inf")), "not finite"), (dict(q=other(5, "bf16"), out=other(5, "bf16")), "5 heads over"),
                         (dict(q=other(4, "f32"), out=other(4, "f32")), "of type bf16 or f16"), (dict(out=other(4, "f16")), "one type and length"),
                         (dict(out=other(4, "bf16", 2)), "one type and length"), (dict(out=q), "takes the queries' place"),
                         (dict(out=other(6, "bf16")), "are wanted"), (dict(kv_lens=array(ctx, [3, 3], "i32")), "kv_lens"),
                         (dict(q_starts=array(ctx, [0], "i32")), "q_starts"), (dict(q_starts=array(ctx, [0.0, 3.0], "f32")), "of type i32"),
                         (dict(page_table=array(ctx, [0, 1], "i32")), "q_starts"),
                         (dict(out=Strided(out, (3, 4, 64), (64, 64, 1), 0)), "overlap"), (dict(q=Strided(q, (3, 4, 64), (-256, 64, 1), 0)), "strides"),
                         (dict(q=Strided(q, (3, 4, 64), (128, 32, 2), 0)), "lie 2 apart")):
        with pytest.raises(capi.TpuHipError, match=says):
            cache.attention(**{**good, **change})
    rows_of = lambda n, dtype="bf16": DeviceArray(ctx, (n, 2, 64), dtype)
    slots = array(ctx, np.arange(5), "i32")
    cache.write(rows_of(5), rows_of(5), slots)
    for k, v, at, says in ((rows_of(5), rows_of(5, "f16"), slots, "one type and length"), (rows_of(5), rows_of(4), slots, "one type and length"),
                           (rows_of(4), rows_of(4), slots, "4] int32"), (rows_of(5, "i32"), rows_of(5), slots, "bf16 or f16 or f32"),
                           (DeviceArray(ctx, (5, 3, 64), "bf16"), rows_of(5), slots, "are wanted"), (rows_of(5), rows_of(5), rows_of(5), "slots"),
                           (Strided(rows_of(5), (5, 2, 64), (-128, 64, 1), 0), rows_of(5), slots, "strides of the keys")):
        with pytest.raises(capi.TpuHipError, match=says):
            cache.write(k, v, at)
    with pytest.raises(capi.TpuHipError, match="rows of the values overlap"):
        cache.read(slots, rows_of(5), Strided(rows_of(5), (5, 2, 64), (64, 64, 1), 0))
    cache.close()


def test_torch_tensors():
    """the cache between torch's own kernels, on torch's stream and on another one, on parts of a tensor: tests/kv_torch.py, in a process of its own,
    since torch has to be imported before the library"""
    res = subprocess.run([sys.executable, os.path.join(os.path.dirname(os.path.abspath(__file__)), "kv_torch.py")], stdout=subprocess.PIPE,
                         stderr=subprocess.STDOUT, text=True, timeout=100)
    assert res.returncode == 0 and res.stdout.strip().endswith("fine"), res.stdout[-3000:]


@pytest.mark.parametrize("bits,n,dim,q_len", [(4, 513, 64, 1), (8, 513, 128, 1), (4, 3000, 64, 3), (4, 300, 160, 40)])
def test_what_cancels_in_a_row_cancels_in_the_result(ctx, bits, n, dim, q_len):
    """float16 results: values that are small between two large ones have large codes and a large offset.  All weights but the first token's are
    alike and their rounding to float16 is as large as it gets, so that it adds up; of the small values that is little"""
    rng = np.random.default_rng(6)
    v = O.rounded(rng.uniform(-0.05, 0.05, (n, 1, dim)), "bf16")
    v[:, :, 0], v[:, :, 1] = -1, 1
    step = float(O.quantise(v, bits)[1][0, 0, 0])
    x = np.linspace(0.5, 1.5, 2001)                              # weights exp(-x) times the step, as far from a float16 number as can be
    product = np.exp(-x) * step
    x = O.rounded(x[np.abs(product.astype(np.float16) / product - 1).argmax()], "bf16").item()
    k = np.zeros((n, 1, dim), np.float32)
    k[1:] = -x
    q = np.zeros((q_len, 2, dim), np.float32)
    q[:, :, 0] = dim ** 0.5 if dim == 64 else 8
    k *= np.float32(dim ** 0.5 / q[0, 0, 0])
    check(ctx, rng, q, [q_len], [O.rounded(k, "bf16")], [v], [n], bits, "f16")


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kv_lens,q_lens,heads,kv_heads,dim", [([513], [1], 8, 2, 128), ([700, 40], [1, 1], 6, 1, 64), ([300], [40], 4, 2, 80),
                                                               ([200, 150], [180, 150], 4, 4, 64), ([2000], [3], 4, 1, 256)])
def test_float16_results_by_the_terms_of_their_rows(ctx, bits, kv_lens, q_lens, heads, kv_heads, dim):
    rng = np.random.default_rng(7)
    k, v = ([rows(rng, n, kv_heads, dim, "bf16", False) for n in kv_lens] for _ in "kv")
    check(ctx, rng, rows(rng, sum(q_lens), heads, dim, "f16", False), q_lens, k, v, kv_lens, bits, "f16")


def test_a_cache_that_there_is_no_memory_for(ctx):
    """is refused, and what comes after it is not"""
    with pytest.raises(capi.TpuHipError) as refused:
        KVCache(ctx, 1 << 20, 64, 256, 8, 32)                    # 1.1 TB
    assert refused.value.status == 3 and "memory" in str(refused.value)
    cache = KVCache(ctx, 2, 2, 64, 4, 32)
    x, slots = array(ctx, np.ones((3, 2, 64)), "bf16"), array(ctx, np.arange(3), "i32")
    with pytest.raises(capi.TpuHipError):
        KVCache(ctx, 1 << 20, 64, 256, 8, 32)
    cache.write(x, x, slots)
    with pytest.raises(capi.TpuHipError):
        KVCache(ctx, 1 << 20, 64, 256, 8, 32)
    cache.read(slots, x, x)
    cache.close()


@pytest.mark.parametrize("far", [1e6, 1e9])
@pytest.mark.parametrize("near", [30, 250, 900])
@pytest.mark.parametrize("bits,dim,heads", [(4, 64, 1), (8, 128, 2), (4, 160, 1), (4, 96, 4)])
def test_large_values_that_some_queries_see_and_larger_ones_that_few_see(ctx, bits, dim, heads, near, far):
    """the first queries' windows hold a value that the others have behind them, and the last ones see tokens `near` times their other ones; all
    with the same weight, so that each of these counts in full"""
    rng = np.random.default_rng(9)
    n, q_len, window = 320, 24, 130
    k, v = (rows(rng, n, 1, dim, "bf16", False) for _ in "kv")
    first = n - q_len
    v[first - window + 3] = O.rounded(v[first - window + 3] * far, "bf16")     # seen by the first three queries
    v[[n - 20, n - 7]] = O.rounded(v[[n - 20, n - 7]] * near, "bf16")
    q = np.zeros((q_len, heads, dim), np.float32)
    check(ctx, rng, q, [q_len], [k], [v], [n], bits, "bf16", window=window)


@pytest.mark.parametrize("bits,heads,dim", [(4, 1, 64), (8, 3, 96), (4, 2, 100), (8, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("seed", range(6))
def test_runs_of_slots_of_every_kind(ctx, bits, heads, dim, seed):
    """pieces in order that begin and end anywhere in a unit, whole units, single slots, slots in reverse and none, one after the other: written and
    read back by other such pieces"""
    rng = np.random.default_rng(seed)
    total = 32 * (40 if seed < 3 else 400)

    def pieces():
        order, at = [], 0
        cuts = rng.choice(np.arange(1, total), rng.integers(1, 60), replace=False)
        cuts = np.unique(np.where(rng.random(len(cuts)) < 0.5, cuts // 32 * 32, cuts))
        parts = [np.arange(a, b) for a, b in zip(np.r_[0, cuts], np.r_[cuts, total]) if a < b]
        parts = [p[::-1] if rng.random() < 0.15 else rng.permutation(p) if rng.random() < 0.15 else p for p in parts]
        rng.shuffle(parts)
        for p in parts:
            order += [np.full(rng.integers(0, 3), -1), p]
        return np.concatenate(order)[:rng.integers(total // 2, total + 40)]

    cache = KVCache(ctx, total // 32, heads, dim, bits, 32)
    to = pieces()
    assert len(np.unique(to[to >= 0])) == (to >= 0).sum()        # each slot once
    x, y = (rows(rng, len(to), heads, dim, "bf16", False) for _ in "kv")
    cache.write(array(ctx, x, "bf16"), array(ctx, y, "bf16"), array(ctx, to, "i32"))
    back = pieces()
    got = [DeviceArray.of(ctx, np.full((len(back), heads, dim), 7.0), "bf16") for _ in range(2)]
    cache.read(array(ctx, back, "i32"), *got)
    for a, b in zip(got, (x, y)):
        held = np.zeros((total + 1, heads, dim), np.float32)     # the last one: of slots that are none
        held[to[to >= 0]] = O.rounded(O.values(b, bits), "bf16")[to >= 0]
        assert np.array_equal(a.numpy(), held[back])
    cache.close()
