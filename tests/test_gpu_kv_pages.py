"""The pages of a batch against a plain list of them; with the cache and attention that they are for."""
import numpy as np
import pytest

import gpu_capture
import mx_oracle as O
from tpu_compiler_amd import capi
from tpu_compiler_amd.kv_cache import DeviceArray, KVPages

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context()
    yield c
    c.close()


def ints(ctx, v):
    return DeviceArray.of(ctx, v, "i32")


class Both:
    """the batch on the device and beside it"""

    def __init__(self, ctx, pages, sequences, max_pages, page):
        self.ctx, self.n = ctx, sequences
        self.here, self.want = KVPages(ctx, pages, sequences, max_pages, page), O.Pages(pages, sequences, max_pages, page)
        self.same()

    def same(self):
        p, w = self.here, self.want
        assert p.lens.numpy().tolist() == w.lens
        assert np.array_equal(p.table.numpy(), w.table())
        assert p.n_free.numpy()[0] == len(w.free) and p.free.numpy()[:len(w.free)].tolist() == w.free

    def grow(self, new, capacity):
        starts, slots, refused = ints(self.ctx, [9] * (self.n + 1)), ints(self.ctx, [9] * (capacity + 3)), ints(self.ctx, [9])
        part = Part(slots, capacity)
        self.here.grow(ints(self.ctx, new), starts, part, refused)
        want = self.want.grow(new, capacity)
        assert starts.numpy().tolist() == want[0]
        assert slots.numpy().tolist() == [int(v) for v in want[1]] + [9] * 3
        assert refused.numpy()[0] == want[2]
        self.same()
        return want

    def trim(self, keep):
        self.here.trim(ints(self.ctx, keep))
        self.want.trim(keep)
        self.same()


class Part:
    def __init__(self, base, n):
        self.base, self.shape, self.dtype = base, (n,), base.dtype

    def data_ptr(self):
        return self.base.data_ptr()

    def stride(self):
        return (1,)


@pytest.mark.parametrize("sequences", [1, 2, 63, 64, 65, 700, 1023, 1024, 1025, 3000])
@pytest.mark.parametrize("page", [32, 96])
def test_sequences_grow_and_shrink(ctx, sequences, page):
    rng = np.random.default_rng(sequences + page)
    b = Both(ctx, sequences * 5, sequences, 12, page)
    refused = 0
    for step in range(12):
        kind = rng.integers(0, 4)
        if kind < 2:
            new = rng.integers(-2, [3, 8 * page][kind], sequences)
            new[rng.random(sequences) < 0.3] = 0
            capacity = int(rng.choice([max(new.clip(0).sum(), 1), new.clip(0).sum() + 40, max(new.clip(0).sum() // 2, 1)]))
            refused += b.grow(new.tolist(), capacity)[2]
        else:
            lens = np.array(b.want.lens)
            keep = np.where(rng.random(sequences) < 0.4, rng.integers(-1, lens + 3), 2 ** 31 - 1)
            b.trim(keep.tolist())
    assert refused or sequences < 3


def test_one_long_sequence(ctx):
    b = Both(ctx, 5000, 1, 5000, 32)
    b.grow([1], 4)
    b.grow([131072], 131072)
    b.grow([0], 0)
    b.grow([5000 * 32 - 131073], 40000)
    assert b.grow([1], 4)[2] == 1                # the row is full
    b.trim([33])
    b.trim([0])
    b.trim([0])


def test_who_gets_pages_when_they_run_out(ctx):
    b = Both(ctx, 4, 5, 4, 32)
    # 1 page, 2 pages, 2 pages that are not there, a page that is no longer free for it, none wanted
    assert b.grow([20, 40, 50, 3, 0], 200)[0] == [0, 20, 60, 60, 60, 60]
    # room in a last page, the last free page, and none for the last one
    assert b.grow([12, 30, 0, 0, 5], 50)[2] == 1
    assert b.want.lens == [32, 70, 0, 0, 0] and not b.want.free
    # the second needs no page, whoever before it gets none
    assert b.grow([1, 24, 0, 0, 0], 50)[0] == [0, 0, 24, 24, 24, 24]
    b.trim([0, 99, 0, 0, 1])
    assert b.grow([0, 1, 0, 0, 0], 0)[2] == 1    # room in its page, but none for its slot
    assert b.grow([0, 1, 0, 0, 0], 1)[2] == 0
    # a row that is not enough takes nothing from those behind it
    c = Both(ctx, 8, 3, 2, 32)
    assert c.grow([65, 64, 10], 74)[0] == [0, 0, 64, 74]
    d = Both(ctx, 8, 3, 2, 32)
    assert d.grow([2 ** 31 - 1, 2 ** 31 - 1, 10], 74)[0] == [0, 0, 0, 10]


def test_what_grew_and_is_taken_off_again_leaves_no_trace(ctx):
    rng = np.random.default_rng(4)
    b = Both(ctx, 900, 100, 30, 64)
    b.grow(rng.integers(0, 300, 100).tolist(), 30000)
    b.trim(rng.integers(0, 200, 100).tolist())
    before, free = list(b.want.lens), b.here.free.numpy().tolist()
    starts, slots, _ = b.grow(rng.integers(0, 300, 100).tolist(), 30000)
    b.trim(before)
    assert b.here.free.numpy().tolist()[:len(b.want.free)] == free[:len(b.want.free)] and b.want.lens == before


def test_arrays_of_the_caller_whose_state_goes_on(ctx):
    table = ints(ctx, [[3, -1, -1, 7, 7], [0, 5, -1, 7, 7]])

    class Rows:
        shape, dtype = (2, 3), "i32"
        data_ptr, stride = staticmethod(table.data_ptr), staticmethod(lambda: (5, 1))

    lens, free, n_free = ints(ctx, [32, 40]), ints(ctx, [1, 2, 4, 6, 0, 0, 0, 0]), ints(ctx, [4])
    p = KVPages(ctx, 8, 2, 3, 32, lens, Rows, free, n_free)
    starts, slots = ints(ctx, [0] * 3), ints(ctx, [0] * 30)
    p.grow(ints(ctx, [2, 25]), starts, slots)
    assert table.numpy().tolist() == [[3, 6, -1, 7, 7], [0, 5, 4, 7, 7]] and lens.numpy().tolist() == [34, 65] and n_free.numpy()[0] == 2
    assert slots.numpy().tolist() == [192, 193] + list(range(168, 192)) + [128] + [-1] * 3
    p.trim(ints(ctx, [99, 0]))
    assert table.numpy().tolist() == [[3, 6, -1, 7, 7], [-1, -1, -1, 7, 7]] and free.numpy().tolist()[:5] == [1, 2, 4, 5, 0]


def test_state_that_is_wrong_is_cut_to_what_there_is(ctx):
    """no length, count or page makes a call touch what is not its own"""
    lens, table = ints(ctx, [-5, 1 << 30, 64]), ints(ctx, [[99, -7, 2], [5, 6, 2 ** 31 - 1], [1, 1, 1]])
    around = ints(ctx, list(range(100, 112)))

    class Free:
        shape, dtype = (8,), "i32"
        data_ptr, stride = staticmethod(lambda: around.data_ptr() + 8), staticmethod(lambda: (1,))

    n_free = ints(ctx, [1000])
    p = KVPages(ctx, 8, 3, 3, 32, lens, table, Free, n_free)
    starts, slots = ints(ctx, [0] * 4), ints(ctx, [0] * 40)
    p.grow(ints(ctx, [10, 10, 10]), starts, slots)
    assert starts.numpy().tolist() == [0, 10, 10, 20]
    assert (slots.numpy() == -1).all()                            # pages 109 and 108 are not there
    p.trim(ints(ctx, [0, 0, 0]))
    p.trim(ints(ctx, [0, 0, 0]))
    assert around.numpy().tolist()[:2] == [100, 101] and around.numpy().tolist()[-2:] == [110, 111]
    assert n_free.numpy()[0] == 8 and not lens.numpy().any()


def test_a_recorded_step_goes_on_by_itself(ctx):
    """the next token of every sequence, recorded once and replayed: pages as a list of them gives them out"""
    sequences, page = 40, 32
    b = Both(ctx, 200, sequences, 5, page)
    rng = np.random.default_rng(0)
    b.grow(rng.integers(0, 100, sequences).tolist(), 5000)
    new, starts, slots, refused = ints(ctx, [1] * sequences), ints(ctx, [0] * (sequences + 1)), ints(ctx, [0] * (sequences + 8)), ints(ctx, [0])
    plan = b.here.plan_grow(new, starts, slots, refused)
    g = gpu_capture.Graph(ctx.h)
    with g.recording():
        plan()
    total = 0
    for step in range(70):
        g.replay()
        want = b.want.grow([1] * sequences, sequences + 8)
        assert slots.numpy().tolist() == [int(v) for v in want[1]] and refused.numpy()[0] == want[2]
        b.same()
        total += want[2]
        if step % 20 == 19:
            b.trim([int(v) for v in rng.integers(0, 90, sequences)])
    g.close()


def test_a_context_s_first_calls_are_recorded():
    """with pages and slots for several workgroups, of which there is one without a counter; later ones by themselves have it"""
    c = capi.Context()
    b = Both(c, 20000, 300, 100, 32)
    rng = np.random.default_rng(5)
    new, starts, slots, refused, keep = ints(c, [0] * 300), ints(c, [0] * 301), ints(c, [0] * 9000), ints(c, [0]), ints(c, [0] * 300)
    trim, grow = b.here.plan_trim(keep), b.here.plan_grow(new, starts, slots, refused)
    g = gpu_capture.Graph(c.h)
    with g.recording():
        trim(), grow()
    for step in range(4):
        for run in (g.replay, lambda: (trim(), grow())):
            stay, more = rng.integers(0, 3000, 300), rng.integers(0, 50, 300)
            c.upload(keep.ptr, stay.astype(np.int32)), c.upload(new.ptr, more.astype(np.int32))
            run()
            b.want.trim(stay.tolist())
            want = b.want.grow(more.tolist(), 9000)
            assert slots.numpy().tolist() == [int(v) for v in want[1]] and refused.numpy()[0] == want[2]
            b.same()
    g.close()
    c.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_the_example_answers_the_same_with_pages_from_the_gpu(ctx, window, sinks):
    """the same pages in the same order: bit for bit"""
    from tpu_compiler_amd import kv_example
    model, rng = kv_example.Model(), np.random.default_rng(8)
    prompts = [rng.integers(0, 512, n) for n in (3, 130, 64, 1)]
    results = [kv_example.generate(ctx, model, prompts, 6, 4, window, sinks, page_tokens=32, pages_on_gpu=g) for g in (False, True)]
    assert results[0][0] == results[1][0] and all(np.array_equal(a, b) for a, b in zip(results[0][1], results[1][1]))


def test_sequences_end_and_others_take_their_pages(ctx):
    """a draft that is not taken, a request that ends, one that comes: rows and attention are those of sequences that never saw the others"""
    from tpu_compiler_amd import kv_example
    rng = np.random.default_rng(2)
    sizes = ctx, 1, 4, 2, 64, 8
    x = {i: rng.standard_normal((300, 8, 64)).astype(np.float32) for i in range(4)}
    parts = lambda i, a, b: np.split(x[i][a:b], [4, 6], 1)

    def step(s, rows):
        """rows[b] = (which text, from, to) of sequence b"""
        s.begin([b - a for _, a, b in rows])
        q, k, v = (np.concatenate(p) for p in zip(*(parts(*r) for r in rows)))
        out = s.attend(0, q, k, v)
        s.end()
        return np.split(out, np.cumsum([b - a for _, a, b in rows])[:-1])

    s = kv_example.SequencesOnGpu(*sizes, 12, 3, 32)
    step(s, [(0, 0, 70), (1, 0, 33), (2, 0, 5)])
    step(s, [(0, 70, 70), (1, 33, 99), (2, 5, 64)])          # six more pages: all twelve but three
    s.trim([70, 40, 0])                                      # a draft is cut, the last one ends
    with pytest.raises(ValueError, match="pages"):
        step(s, [(0, 70, 71), (1, 40, 41), (3, 0, 300)])
    assert s.lens == [70, 40, 0]
    got = step(s, [(0, 70, 73), (1, 40, 41), (3, 0, 160)])
    s.close()
    for which, a, b in ((0, 70, 73), (1, 40, 41), (3, 0, 160)):
        alone = kv_example.Sequences(*sizes, 10, 32)
        if a:
            step(alone, [(which, 0, a)])
        want = step(alone, [(which, a, b)])[0]
        alone.close()
        # the same rows; sums may be shared otherwise: two roundings of a bfloat16 number of size three at most, and of weights (2^-11 of each)
        assert np.abs(got.pop(0) - want).max() <= 2.0 ** -5
