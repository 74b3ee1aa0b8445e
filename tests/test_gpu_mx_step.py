"""A step of a language model from its operators on one stream: drafts taken back, pages for new tokens, products, rows written to the cache, attention,
products again.  Recorded once and replayed, it goes on by itself: the host writes its inputs and reads its results, nothing else."""
import numpy as np
import pytest

import gpu_capture
import kv_bounds
import mx_oracle as O
from tpu_compiler_amd import capi, mx
from tpu_compiler_amd.kv_cache import DeviceArray, KVCache, KVPages

pytestmark = pytest.mark.gpu
SEQUENCES, CAPACITY, PAGES, MOST, PAGE = 5, 20, 20, 4, 32
HEADS, KV_HEADS, DIM, WIDTH, BITS = 4, 2, 64, 256, 8


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context()
    yield c
    c.close()


class Heads:
    """columns of an array's rows as heads"""

    def __init__(self, base, first, heads):
        self.base, self.first, self.shape, self.dtype = base, first, (base.shape[0], heads, DIM), base.dtype

    def data_ptr(self):
        return self.base.data_ptr() + 2 * self.first * DIM

    def stride(self):
        return self.base.shape[1], DIM, 1


class Step:
    def __init__(self, ctx, qkv_w, out_w):
        zeros = lambda shape, dtype: DeviceArray.of(ctx, np.zeros(shape), dtype)
        self.ctx, self.pages, self.cache = ctx, KVPages(ctx, PAGES, SEQUENCES, MOST, PAGE), KVCache(ctx, PAGES, KV_HEADS, DIM, BITS, PAGE)
        self.new, self.keep = zeros(SEQUENCES, "i32"), zeros(SEQUENCES, "i32")
        self.starts, self.slots, self.refused = zeros(SEQUENCES + 1, "i32"), zeros(CAPACITY, "i32"), zeros(1, "i32")
        self.x, self.qkv = zeros((CAPACITY, WIDTH), "bf16"), zeros((CAPACITY, (HEADS + 2 * KV_HEADS) * DIM), "bf16")
        self.seen, self.out = zeros((CAPACITY, HEADS * DIM), "bf16"), zeros((CAPACITY, WIDTH), "bf16")
        q, k, v = (Heads(self.qkv, first, n) for first, n in ((0, HEADS), (HEADS, KV_HEADS), (HEADS + KV_HEADS, KV_HEADS)))
        p = self.pages
        self.calls = [p.plan_trim(self.keep), p.plan_grow(self.new, self.starts, self.slots, self.refused), mx.plan_product(ctx, self.x, qkv_w, self.qkv),
                      self.cache.plan_write(k, v, self.slots),
                      self.cache.plan_attention(q, Heads(self.seen, 0, HEADS), self.starts, p.lens, p.table, max_q=CAPACITY, max_kv=MOST * PAGE),
                      mx.plan_product(ctx, self.seen, out_w, self.out, residual=self.x)]

    def __call__(self):
        for call in self.calls:
            call()

    def give(self, new, keep, x):
        for a, values in ((self.new, new), (self.keep, keep)):
            self.ctx.upload(a.ptr, np.array(values, np.int32))
        self.ctx.upload(self.x.ptr, (x.view(np.uint32) >> 16).astype(np.uint16))

    def state(self):
        p = self.pages
        return [a.numpy() for a in (p.lens, p.table, p.n_free, self.starts, self.slots, self.refused, self.qkv, self.seen, self.out)]


def test_a_recorded_step_of_a_model_goes_on_by_itself(ctx):
    rng = np.random.default_rng(0)
    weights = [O.rounded(rng.standard_normal(s) / 16, "f32") for s in (((HEADS + 2 * KV_HEADS) * DIM, WIDTH), (WIDTH, HEADS * DIM))]
    qkv_w, out_w = (mx.MXMatrix(ctx, *w.shape).quantize(DeviceArray.of(ctx, w, "f32")) for w in weights)
    qkv_v, out_v = (O.values(*O.quantized(w), w.shape[1]) for w in weights)
    recorded, beside, pages = Step(ctx, qkv_w, out_w), Step(ctx, qkv_w, out_w), O.Pages(PAGES, SEQUENCES, MOST, PAGE)
    texts = [[np.zeros((0, KV_HEADS, DIM))] * 2 for _ in range(SEQUENCES)]
    g = gpu_capture.Graph(ctx.h)
    with g.recording():
        recorded()
    refused = cut = 0
    for step in range(24):
        lens = list(pages.lens)
        keep = [int(n if rng.random() < 0.6 else max(0, n - rng.integers(0, 6))) for n in lens]
        if step % 8 == 7:
            keep[step % SEQUENCES] = 0                                   # a request ends
        new = [int(n) for n in rng.integers(0, 7, SEQUENCES)]            # more than there is room for, now and then
        x = O.rounded(rng.standard_normal((CAPACITY, WIDTH)), "bf16")
        for s in (recorded, beside):
            s.give(new, keep, x)
        g.replay()
        got = recorded.state()
        beside()
        pages.trim(keep)
        starts, slots, short = pages.grow(new, CAPACITY)
        refused, cut = refused + short, cut + (keep != lens)
        total = starts[-1]
        for i, (a, b) in enumerate(zip(got, beside.state())):
            rows = total if i == 7 else len(a)                           # attention leaves rows behind the last sequence as they were
            assert np.array_equal(a[:rows], b[:rows]), (step, i)
        assert got[0].tolist() == pages.lens and np.array_equal(got[1], pages.table()) and got[2][0] == len(pages.free)
        assert got[3].tolist() == starts and got[4].tolist() == [int(v) for v in slots] and got[5][0] == short
        qkv, seen, out = (v.astype(np.float64) for v in got[6:])
        want, size = O.product(O.values(*O.quantized(x), WIDTH), qkv_v)
        assert (np.abs(qkv - want) <= O.bound(want, size, WIDTH, "bf16")).all()
        q, k, v = np.split(qkv.reshape(CAPACITY, -1, DIM), [HEADS, HEADS + KV_HEADS], 1)
        for i, (a, b) in enumerate(zip(starts, starts[1:])):
            texts[i] = [np.concatenate([text[:keep[i]], rows[a:b]]) for text, rows in zip(texts[i], (k, v))]
        want, limit = kv_bounds.attention(q[:total], [t[0] for t in texts], [t[1] for t in texts], BITS, np.diff(starts), pages.lens, DIM ** -0.5, "bf16")
        assert (np.abs(seen[:total].reshape(total, HEADS, DIM) - want) <= limit).all()
        want, size = O.product(O.values(*O.quantized(seen[:total]), HEADS * DIM), out_v, None, x[:total].astype(np.float64))
        assert (np.abs(out[:total] - want) <= O.bound(want, size, HEADS * DIM, "bf16")).all()
    assert refused and cut
    g.close()
    for s in (recorded, beside):
        s.cache.close()
