"""Attention to the key/value cache, token by token: inputs (kv_marks) of which every token seen, and no other, shows in the result, at
lengths that are split over waves and workgroups and joined again."""
import numpy as np
import pytest

import gpu_capture
import kv_marks as M
import kv_oracle as O
from test_gpu_kv_cache import Sequences, array, ctx, rows  # noqa: F401 (a fixture)
from tpu_compiler_amd.kv_cache import DeviceArray

pytestmark = pytest.mark.gpu

# (tokens, queries, heads, kv_heads, window, sinks): single tokens of one unit to thousands, in splits that the last workgroup joins and in more;
# a few; prompts with so few and so many rows that each form of the kernel has its turn; windows and first tokens at and beside units' edges
CASES = [([1, 33, 700], [1, 1, 1], 8, 2, 0, 0), ([9000], [1], 16, 1, 0, 0), ([4000, 129, 64], [1, 1, 1], 24, 3, 0, 0), ([40000], [1], 32, 2, 0, 0),
         ([2500, 40], [5, 3], 20, 5, 0, 0), ([4100], [40], 4, 1, 0, 0), ([300, 7], [300, 7], 4, 2, 0, 0), ([1100], [700], 32, 8, 0, 0),
         ([500, 400], [500, 390], 64, 32, 0, 0), ([100] * 6, [80] * 6, 64, 16, 0, 0),
         ([610, 33, 5], [1, 1, 1], 8, 2, 100, 0), ([6000], [1], 8, 2, 4000, 5), ([6000, 900], [1, 1], 8, 1, 64, 32), ([777], [1], 4, 4, 31, 33),
         ([900], [9], 12, 4, 65, 4), ([1500, 200], [300, 200], 8, 2, 130, 17), ([2000], [600], 64, 16, 33, 1), ([650], [650], 32, 8, 2, 0)]


@pytest.mark.parametrize("bits,dim,dtype", [(4, 128, "f16"), (8, 64, "f16"), (4, 256, "f16"), (8, 80, "bf16"), (4, 160, "f16")])
@pytest.mark.parametrize("case", CASES)
def test_each_token_counts_once(ctx, case, bits, dim, dtype):
    kv_lens, q_lens, heads, kv_heads, window, sinks = case
    rng = np.random.default_rng(len(kv_lens))
    v = M.counting(kv_lens, kv_heads, dim, bits)
    s = Sequences(ctx, rng, kv_lens, kv_heads, dim, bits, 32, k=[rows(rng, n, kv_heads, dim, "bf16", False) for n in kv_lens], v=v)
    got = s.attend(rows(rng, sum(q_lens), heads, dim, dtype, False), q_lens, dtype, scale=0.0, window=window, sinks=sinks)
    s.cache.close()
    want = M.counted(kv_lens, q_lens, dim, bits, window, sinks)[:, None]
    assert (np.abs(got - want) <= M.counting_limit(want, dtype)).all()


def test_each_of_131072_tokens_counts_once(ctx):
    n, dim = 131072, 256
    rng = np.random.default_rng(0)
    s = Sequences(ctx, rng, [n], 1, dim, 4, 128, k=[np.zeros((n, 1, dim), np.float32)], v=M.counting([n], 1, dim, 4))
    for q_len in (1, 4):
        for heads in (8, 16):
            got = s.attend(rows(rng, q_len, heads, dim, "f16", False), [q_len], "f16", scale=0.0)
            want = M.counted([n], [q_len], dim, 4)[:, None]
            assert (np.abs(got - want) <= M.counting_limit(want, "f16")).all()
    s.cache.close()


@pytest.mark.parametrize("bits,dim,dtype", [(4, 128, "f16"), (8, 64, "f16"), (4, 72, "bf16"), (8, 200, "f16")])
@pytest.mark.parametrize("case", CASES)
def test_a_token_that_is_looked_for_is_found(ctx, case, bits, dim, dtype):
    kv_lens, q_lens, heads, kv_heads, window, sinks = case
    rng = np.random.default_rng(sum(kv_lens))
    q, k, v, scale = M.finding(rng, kv_lens, q_lens, heads, kv_heads, dim, bits, window, sinks)
    s = Sequences(ctx, rng, kv_lens, kv_heads, dim, bits, 64, k=k, v=v)
    got = s.attend(q, q_lens, dtype, scale=scale, window=window, sinks=sinks)
    s.cache.close()
    want = M.found(q, k, v, bits, q_lens, kv_lens, scale, window, sinks)
    assert (np.abs(got - want) <= M.finding_limit(want, dtype)).all()


def test_a_recorded_step_finds_the_token_it_writes(ctx):
    """a replay whose lengths or slots were those of the recording would find another"""
    rng = np.random.default_rng(1)
    heads, d, page, lens = 2, 64, 32, [3000, 45]
    q, k, v, scale = M.finding(rng, [n + 4 for n in lens], [4, 4], 4, heads, d, 4)
    s = Sequences(ctx, rng, lens, heads, d, 4, page, k=[x[:n] for x, n in zip(k, lens)], v=[x[:n] for x, n in zip(v, lens)])
    extra = [array(ctx, np.zeros((2, heads, d)), "bf16") for _ in range(2)]
    qs, out = array(ctx, np.zeros((2, 4, d)), "bf16"), DeviceArray(ctx, (2, 4, d), "bf16")
    slots, held = array(ctx, [-1, -1], "i32"), array(ctx, lens, "i32")
    write = s.cache.plan_write(*extra, slots)
    attend = s.cache.plan_attention(qs, out, array(ctx, [0, 1, 2], "i32"), held, array(ctx, s.table, "i32"), max_q=1, max_kv=3008)
    write(), attend()
    graph = gpu_capture.Graph(ctx.h)
    with graph.recording():
        write()
        attend()
    as_bf16 = lambda x: (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    for step in range(4):
        at = [n + step for n in lens]
        for x, new in zip(extra, (k, v)):
            ctx.upload(x.ptr, as_bf16(np.stack([y[t] for y, t in zip(new, at)])))
        pattern = np.stack([np.repeat(np.where(y[t] > 0, 1.0, -1.0), 2, 0) for y, t in zip(k, at)])     # the queries are the new token's pattern
        ctx.upload(qs.ptr, as_bf16(pattern))
        ctx.upload(slots.ptr, np.array([s.table[i][t // page] * page + t % page for i, t in enumerate(at)], np.int32))
        ctx.upload(held.ptr, np.array([t + 1 for t in at], np.int32))
        graph.replay()
        got = out.numpy().astype(np.float64)
        want = np.stack([np.repeat(O.values(y[t], 4), 2, 0) for y, t in zip(v, at)])
        assert (np.abs(got - want) <= M.finding_limit(want, "bf16")).all()
        attend()
        assert np.array_equal(out.numpy(), got.astype(np.float32))
    graph.close()
    s.cache.close()
