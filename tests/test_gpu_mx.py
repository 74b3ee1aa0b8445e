"""Microscaled 4-bit numbers and their products against their definitions in 64 bits."""
import numpy as np
import pytest

import gpu_capture
import mx_oracle as O
from tpu_compiler_amd import capi, mx
from tpu_compiler_amd.kv_cache import DeviceArray

pytestmark = pytest.mark.gpu
SIZES = {"bf16": 2, "f16": 2, "f32": 4, "u8": 1}


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context()
    yield c
    c.close()


class Part:
    """rows of a part of a larger array, `first` elements from its beginning"""

    def __init__(self, base, shape, stride, first=0):
        self.base, self.shape, self._stride, self.dtype, self.first = base, shape, stride, base.dtype, first

    def data_ptr(self):
        return self.base.data_ptr() + self.first * SIZES[self.dtype]

    def stride(self):
        return self._stride


def part_of(ctx, values, dtype, extra, first, fill=7):
    """the values as rows `extra` elements longer than they are wide -> (the part, the whole array)"""
    rows, cols = values.shape
    host = np.full(rows * (cols + extra) + first, fill, np.float64)
    at = first + np.arange(rows)[:, None] * (cols + extra) + np.arange(cols)
    host[at] = values
    base = DeviceArray.of(ctx, host, dtype)
    return Part(base, (rows, cols), (cols + extra, 1), first), base


def spread(rng, rows, cols, dtype):
    """numbers of all sizes, blocks of different ones"""
    x = rng.standard_normal((rows, cols)) * 10.0 ** rng.integers(-3, 4, (rows, 1)) * 2.0 ** rng.integers(-4, 5, (1, cols))
    return O.rounded(x, dtype)


def quantised(ctx, x, dtype):
    m = mx.MXMatrix(ctx, *x.shape)
    return m.quantize(DeviceArray.of(ctx, x, dtype))


def codes_of(rng, rows, cols, low, high):
    """codes and scales of any kind; zeros behind the last column"""
    blocks = -(-cols // 32)
    c = rng.integers(0, 16, (rows, blocks * 32)).astype(np.uint8)
    c[:, cols:] = 0
    return c[:, 0::2] | c[:, 1::2] << 4, rng.integers(low, high + 1, (rows, blocks)).astype(np.uint8)


def matrix(ctx, codes, scales, cols):
    return mx.MXMatrix(ctx, codes.shape[0], cols, DeviceArray.of(ctx, codes, "u8"), DeviceArray.of(ctx, scales, "u8"))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (7, 100), (1, 4096), (33, 257), (130, 1000), (3, 5000), (2, 20001)])
def test_rows_are_quantised_and_read_back(ctx, dtype, rows, cols):
    x = spread(np.random.default_rng(rows * cols), rows, cols, dtype)
    m = quantised(ctx, x, dtype)
    codes, scales = O.quantized(x)
    assert np.array_equal(m.codes.numpy(), codes) and np.array_equal(m.scales.numpy(), scales)
    for to in ("bf16", "f16", "f32"):
        out = DeviceArray(ctx, x.shape, to)
        m.read(out)
        assert np.array_equal(out.numpy().astype(np.float32), O.rounded(O.values(codes, scales, cols), to), equal_nan=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("extra,first", [(1, 0), (0, 1), (3, 5), (64, 0)])
def test_rows_of_longer_ones_are_quantised_and_nothing_beside_them_is_written(ctx, dtype, extra, first):
    x = spread(np.random.default_rng(extra * 8 + first), 6, 75, dtype)
    a, _ = part_of(ctx, x, dtype, extra, first)
    codes, scales = O.quantized(x)
    # a matrix whose rows are parts of longer ones too
    c, s = (DeviceArray.of(ctx, np.full((6, n), 9), "u8") for n in (96, 11))
    m = mx.MXMatrix(ctx, 6, 75, Part(c, (6, 48), (96, 1), 32), Part(s, (6, 3), (11, 1), 5))
    m.quantize(a)
    want_c, want_s = np.full((6, 96), 9, np.uint8), np.full((6, 11), 9, np.uint8)
    want_c[:, 32:80], want_s[:, 5:8] = codes, scales
    assert np.array_equal(c.numpy(), want_c) and np.array_equal(s.numpy(), want_s)
    out, base = part_of(ctx, np.zeros((6, 75)), dtype, extra, first)
    before = base.numpy()
    m.read(out)
    at = first + np.arange(6)[:, None] * (75 + extra) + np.arange(75)
    before[at] = O.rounded(O.values(codes, scales, 75), dtype)
    assert np.array_equal(base.numpy(), before)


def test_ties_largest_and_smallest_numbers(ctx):
    """every middle between two codes, its neighbours, sizes beyond the largest code, at scales from the smallest to the largest, both signs"""
    rows = []
    for e in (-149, -140, -130, -127, -126, -125, -124, -20, 0, 1, 60, 124, 125):
        for top in (4.0, 5.0, 6.0, 7.0, 7.9990234375):
            base = np.array([top, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0, 0.0625, 6.5], np.float32)
            base = np.minimum(base, np.float32(top))
            with np.errstate(over="ignore", under="ignore"):
                v = (base.astype(np.float64) * 2.0 ** e).astype(np.float32)
                v = np.concatenate([v, np.nextafter(v[1:9], np.float32(np.inf)), np.nextafter(v[1:9], np.float32(0))])
            v = np.where(np.abs(v) > np.abs(v[0]), v[0], v)
            rows += [np.pad(v, (0, 32 - len(v))), np.pad(-v, (0, 32 - len(v)))]
    x = np.array(rows, np.float32)
    assert np.isfinite(x).all()
    for dtype in ("f32", "bf16", "f16"):
        part = O.rounded(x, dtype)
        part = np.where(np.isfinite(part), part, np.float32(1))
        m = quantised(ctx, part, dtype)
        codes, scales = O.quantized(part)
        assert np.array_equal(m.codes.numpy(), codes) and np.array_equal(m.scales.numpy(), scales)
        out = DeviceArray(ctx, x.shape, "f32")
        m.read(out)
        assert np.array_equal(out.numpy(), O.values(codes, scales, 32).astype(np.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_block_that_holds_no_number_is_nan_and_no_other(ctx, dtype, bad):
    x = spread(np.random.default_rng(1), 4, 200, dtype)
    x[1, 40] = bad
    x[2, 199] = bad
    m = quantised(ctx, x, dtype)
    codes, scales = O.quantized(x)
    assert np.array_equal(m.codes.numpy(), codes) and np.array_equal(m.scales.numpy(), scales)
    out = DeviceArray(ctx, x.shape, dtype)
    m.read(out)
    got = out.numpy()
    assert np.isnan(got[1, 32:64]).all() and np.isnan(got[2, 192:]).all() and np.isnan(got).sum() == 40


def test_every_code_and_scale_is_read_as_it_stands(ctx):
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, 1)
    m = matrix(ctx, codes, scales, 512)
    for to in ("bf16", "f16", "f32"):
        out = DeviceArray(ctx, (256, 512), to)
        m.read(out)
        with np.errstate(over="ignore"):
            want = O.rounded(O.values(codes, scales, 512), to)
        assert np.array_equal(out.numpy().astype(np.float32), want, equal_nan=True)


SHAPES = [(1, 1, 1), (1, 32, 16), (1, 4096, 100), (2, 33, 17), (3, 512, 1000), (5, 2050, 33), (8, 4096, 130), (4, 8197, 40), (16, 2000, 50),
          (16, 100, 64), (17, 64, 65), (31, 1000, 130), (48, 4096, 48), (64, 512, 257), (65, 300, 64), (130, 2050, 70), (200, 640, 333),
          (257, 1024, 512), (300, 2080, 999)]


@pytest.mark.parametrize("rows,cols,n", SHAPES)
def test_sums_that_32_bits_hold_come_out_as_they_are(ctx, rows, cols, n):
    """products are multiples of 2^-2 up to 36, times up to four powers of two: below 2^24 of the smallest for 4096 columns"""
    rng = np.random.default_rng(rows + cols + n)
    x, w = codes_of(rng, rows, cols, 127, 128), codes_of(rng, n, cols, 126, 127)
    want, size = O.product(O.values(*x, cols), O.values(*w, cols))
    assert size.max() < 2.0 ** 24 / 8
    out = DeviceArray.of(ctx, np.full((rows, n), 7.0), "f32")
    mx.product(ctx, matrix(ctx, *x, cols), matrix(ctx, *w, cols), out)
    assert np.array_equal(out.numpy(), want)


# sizes that take tiles of each size; sums of 256 numbers and of several times as many, whole and with a rest
@pytest.mark.parametrize("rows,n,cols", [(rows, n, cols) for cols in (256, 512, 600, 768, 1024, 1250, 2304)
                                         for rows, n in ((60, 1000), (250, 4096), (500, 4090), (770, 4096), (512, 16380), (2048, 8190))
                                         if rows * n * cols < 2 ** 34.5])
def test_tiles_of_every_size_come_out_as_they_are_each_time(ctx, rows, cols, n):
    rng = np.random.default_rng(rows + cols + n)
    x, w = codes_of(rng, rows, cols, 127, 128), codes_of(rng, n, cols, 126, 127)
    xv, wv = O.values(*x, cols).astype(np.float32), O.values(*w, cols).astype(np.float32)
    assert cols * 72 < 2 ** 24 / 8                     # in units of 2^-3, in any order
    want = xv @ wv.T
    a, b = matrix(ctx, *x, cols), matrix(ctx, *w, cols)
    for _ in range(3):
        out = DeviceArray.of(ctx, np.full((rows, n), 7.0), "f32")
        mx.product(ctx, a, b, out)
        assert np.array_equal(out.numpy(), want)
        out.free()
    for m in (a, b):
        m.free()


# a few rows, short sums into many columns: waves in two, four and eight groups, a last column that leaves some without
@pytest.mark.parametrize("rows,cols", [(1, 40), (3, 512), (16, 224), (2, 700), (1, 1500), (5, 2048), (4, 2040)])
@pytest.mark.parametrize("n", [8193, 16400, 20001, 33000, 65541])
def test_few_rows_into_many_columns(ctx, rows, cols, n):
    x, w, out, want = whole_numbers(ctx, rows, cols, n, n + cols)
    mx.product(ctx, x, w, out)
    assert np.array_equal(out.numpy(), want)
    values = DeviceArray(ctx, (rows, cols), "f32")
    x.read(values)
    mx.product(ctx, values, w, out, residual=out)      # blocks' largest numbers may be too small for a scale of 1: still the same values
    assert np.array_equal(out.numpy(), 2 * want)


# long sums, shared by workgroups
@pytest.mark.parametrize("rows,cols,n", [(1, 16384, 100), (2, 20000, 64), (17, 16384, 200), (40, 16384, 1000), (64, 8192, 4096), (128, 16384, 2048), (16, 30000, 512)])
def test_long_sums(ctx, rows, cols, n):
    rng = np.random.default_rng(cols)
    x, w = codes_of(rng, rows, cols, 127, 127), codes_of(rng, n, cols, 127, 127)
    want, _ = O.product(O.values(*x, cols), O.values(*w, cols))
    assert cols * 36 < 2 ** 24 / 4
    a, b = matrix(ctx, *x, cols), matrix(ctx, *w, cols)
    for _ in range(3):
        out = DeviceArray.of(ctx, np.full((rows, n), 7.0), "f32")
        mx.product(ctx, a, b, out)
        assert np.array_equal(out.numpy(), want)


# sizes that take the tiles between the smallest and the largest, and parts of them; sums with a whole number of parts and of pieces, and with a rest
@pytest.mark.parametrize("rows,cols,n", [(514, 16384, 500), (514, 16600, 500), (640, 32768, 200), (1921, 4096, 1000), (1921, 4400, 1000), (1543, 1250, 2048),
                                         (1543, 1600, 2048), (1606, 16384, 1000), (1606, 16900, 1000), (1158, 520, 2048), (1795, 16384, 1000), (1795, 16900, 1000),
                                         (1543, 300, 5000), (1600, 1100, 5001), (2054, 700, 2048), (1795, 300, 8190)])
def test_tiles_and_parts_with_a_residual_and_what_is_no_number(ctx, rows, cols, n):
    """a NaN block of x in its last row and one of w in the middle: their row and column, and nothing else"""
    rng = np.random.default_rng(rows + cols)
    x, w = codes_of(rng, rows, cols, 127, 127), codes_of(rng, n, cols, 127, 127)
    want = O.values(*x, cols).astype(np.float32) @ O.values(*w, cols).astype(np.float32).T
    more = rng.integers(-1000, 1000, (rows, n)).astype(np.float32)
    assert cols * 36 < 2 ** 24 / 4 - 1000              # in units of 2^-2, in any order
    want += more
    x[1][rows - 1, -1] = w[1][n // 2, 0] = 255
    want[rows - 1] = want[:, n // 2] = np.nan
    a, b, out = matrix(ctx, *x, cols), matrix(ctx, *w, cols), DeviceArray(ctx, (rows, n), "f32")
    for _ in range(2):
        ctx.upload(out.ptr, more)
        mx.product(ctx, a, b, out, residual=out)
        assert np.array_equal(out.numpy(), want, equal_nan=True)
    for m in (a, b, out):
        m.free()


@pytest.mark.parametrize("ready", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,n", SHAPES)
def test_products_of_rows(ctx, rows, cols, n, dtype, ready):
    rng = np.random.default_rng(rows * cols + n)
    x = O.rounded(rng.standard_normal((rows, cols)) * 2.0 ** rng.integers(-3, 4, (1, cols)), dtype)
    w = codes_of(rng, n, cols, 118, 124)
    bias = O.rounded(rng.standard_normal(n), "f32") if n % 2 else None
    residual = O.rounded(rng.standard_normal((rows, n)), dtype) if rows % 2 or n % 2 == 0 else None
    want, size = O.product(O.values(*O.quantized(x), cols), O.values(*w, cols), bias, residual)
    out = DeviceArray.of(ctx, np.full((rows, n), 7.0), dtype)
    a = DeviceArray.of(ctx, x, dtype)
    mx.product(ctx, quantised(ctx, x, dtype) if ready else a, matrix(ctx, *w, cols), out, None if bias is None else DeviceArray.of(ctx, bias, "f32"),
               None if residual is None else DeviceArray.of(ctx, residual, dtype))
    off = np.abs(out.numpy().astype(np.float64) - want)
    assert (off <= O.bound(want, size, cols, dtype)).all(), (off / O.bound(want, size, cols, dtype)).max()


@pytest.mark.parametrize("rows,cols,n", [(1, 100, 37), (5, 600, 130), (70, 513, 66), (300, 1056, 200)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_of_longer_ones_and_a_residual_in_place(ctx, rows, cols, n, dtype):
    rng = np.random.default_rng(n)
    x, y = O.rounded(rng.standard_normal((rows, cols)), dtype), O.rounded(rng.standard_normal((rows, n)), dtype)
    blocks = -(-cols // 32)
    w = codes_of(rng, n, cols, 120, 124)
    c, s = (DeviceArray.of(ctx, np.pad(v, ((0, 0), (p, q)), constant_values=255), "u8") for v, p, q in ((w[0], 16, 32), (w[1], 1, 2)))
    w_m = mx.MXMatrix(ctx, n, cols, Part(c, (n, blocks * 16), (blocks * 16 + 48, 1), 16), Part(s, (n, blocks), (blocks + 3, 1), 1))
    a, _ = part_of(ctx, x, dtype, 9, 1, fill=np.nan)
    out, base = part_of(ctx, y, dtype, 5, 3)
    before = base.numpy().astype(np.float64)
    mx.product(ctx, a, w_m, out, residual=out)
    want, size = O.product(O.values(*O.quantized(x), cols), O.values(*w, cols), None, y)
    got = base.numpy().astype(np.float64)
    at = 3 + np.arange(rows)[:, None] * (n + 5) + np.arange(n)
    assert (np.abs(got[at] - want) <= O.bound(want, size, cols, dtype)).all()
    beside = np.ones(len(got), bool)
    beside[at] = False
    assert np.array_equal(got[beside], before[beside])


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_nan_and_far_apart_scales_stay_where_they_are(ctx, rows):
    rng = np.random.default_rng(5)
    cols, n = 700, 90
    x, w = codes_of(rng, rows, cols, 90, 160), codes_of(rng, n, cols, 90, 160)
    x[1][2, 3], w[1][11, 21], w[1][89, 0] = 255, 255, 255
    xv, wv = O.values(*x, cols), O.values(*w, cols)
    want, size = O.product(np.nan_to_num(xv), np.nan_to_num(wv))
    out = DeviceArray(ctx, (rows, n), "f32")
    mx.product(ctx, matrix(ctx, *x, cols), matrix(ctx, *w, cols), out)
    got = out.numpy().astype(np.float64)
    nan = np.zeros((rows, n), bool)
    nan[2] = nan[:, 11] = nan[:, 89] = True
    assert np.array_equal(np.isnan(got), nan)
    assert (np.abs(got - want) <= O.bound(want, size, cols, "f32"))[~nan].all()


@pytest.mark.parametrize("rows,cols,n", [(1, 2048, 256), (6, 2048, 1000), (64, 1024, 512), (100, 4096, 64), (500, 512, 512)])
def test_a_recorded_product_follows_its_inputs(ctx, rows, cols, n):
    """replayed several times with the context's own work in between; the same bits as the call by itself, each time"""
    rng = np.random.default_rng(3)
    w = matrix(ctx, *codes_of(rng, n, cols, 120, 124), cols)
    x, out = DeviceArray.of(ctx, np.zeros((rows, cols)), "bf16"), DeviceArray(ctx, (rows, n), "bf16")
    plan = mx.plan_product(ctx, x, w, out)
    plan()
    g = gpu_capture.Graph(ctx.h)
    with g.recording():
        plan()
    other, much = DeviceArray(ctx, (rows, n), "bf16"), DeviceArray(ctx, (300, n), "f32")
    more = quantised(ctx, O.rounded(rng.standard_normal((300, cols)), "bf16"), "bf16")
    for _ in range(4):
        v = O.rounded(rng.standard_normal((rows, cols)), "bf16")
        b = (v.view(np.uint32) >> 16).astype(np.uint16)
        ctx.upload(x.ptr, b)
        g.replay()
        got = out.numpy()
        mx.product(ctx, more, w, much)
        mx.product(ctx, x, w, other)
        assert np.array_equal(got, other.numpy())
        want, size = O.product(O.values(*O.quantized(v), cols), O.values(w.codes.numpy(), w.scales.numpy(), cols))
        assert (np.abs(got - want) <= O.bound(want, size, cols, "bf16")).all()
    g.close()


@pytest.mark.parametrize("x_type,dtype", [("f32", "bf16"), ("bf16", "f32"), ("f16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("rows", [2, 70])
def test_rows_of_one_type_and_results_of_another(ctx, rows, x_type, dtype):
    rng, cols, n = np.random.default_rng(rows), 700, 75
    x, more = O.rounded(rng.standard_normal((rows, cols)), x_type), O.rounded(rng.standard_normal((rows, n)), dtype)
    w = codes_of(rng, n, cols, 118, 124)
    want, size = O.product(O.values(*O.quantized(x), cols), O.values(*w, cols), None, more)
    out = DeviceArray.of(ctx, more, dtype)
    mx.product(ctx, DeviceArray.of(ctx, x, x_type), matrix(ctx, *w, cols), out, residual=out)
    assert (np.abs(out.numpy().astype(np.float64) - want) <= O.bound(want, size, cols, dtype)).all()


def whole_numbers(ctx, rows, cols, n, seed):
    """operands and their product, which 32 bits hold in any order"""
    rng = np.random.default_rng(seed)
    x, w = codes_of(rng, rows, cols, 127, 127), codes_of(rng, n, cols, 127, 127)
    assert cols * 36 < 2 ** 24 / 4
    want, _ = O.product(O.values(*x, cols), O.values(*w, cols))
    return matrix(ctx, *x, cols), matrix(ctx, *w, cols), DeviceArray.of(ctx, np.full((rows, n), 7.0), "f32"), want


def test_two_contexts_at_once():
    """sums in parts on two streams: each context has counters and parts of its own"""
    contexts = [capi.Context(), capi.Context()]
    cases = [[(c,) + whole_numbers(c, rows, 16384, n, n) for rows, n in ((64, 500), (17, 300))] for c in contexts]
    plans = [mx.plan_product(c, x, w, out) for pair in zip(*cases) for c, x, w, out, _ in pair]
    for _ in range(10):
        for plan in plans:
            plan()
    for case in cases:
        for c, _, _, out, want in case:
            assert np.array_equal(out.numpy(), want)
    for c in contexts:
        c.close()


def test_a_context_s_first_call_is_recorded():
    """no memory for parts then, which later calls of the context by themselves have"""
    c = capi.Context()
    x, w, out, want = whole_numbers(c, 40, 16384, 300, 1)
    plan = mx.plan_product(c, x, w, out)
    g = gpu_capture.Graph(c.h)
    with g.recording():
        plan()
    for _ in range(3):
        c.upload(out.ptr, np.zeros((40, 300), np.float32))
        g.replay()
        assert np.array_equal(out.numpy(), want)
        c.upload(out.ptr, np.zeros((40, 300), np.float32))
        plan()
        assert np.array_equal(out.numpy(), want)
    g.close()
    c.close()


def test_the_same_call_gives_the_same_bits(ctx):
    rng = np.random.default_rng(9)
    for rows, cols, n in ((1, 4096, 512), (16, 16384, 64), (60, 8192, 128), (128, 4096, 256)):
        x, w = matrix(ctx, *codes_of(rng, rows, cols, 100, 150), cols), matrix(ctx, *codes_of(rng, n, cols, 100, 150), cols)
        results = []
        for _ in range(5):
            out = DeviceArray.of(ctx, np.zeros((rows, n)), "f32")
            mx.product(ctx, x, w, out)
            results.append(out.numpy())
        assert all(np.array_equal(results[0], r) for r in results)


def test_no_rows(ctx):
    w = matrix(ctx, *codes_of(np.random.default_rng(0), 5, 64, 120, 124), 64)
    empty, out = DeviceArray(ctx, (0, 64), "bf16"), DeviceArray(ctx, (0, 5), "bf16")
    mx.product(ctx, empty, w, out)
    mx.product(ctx, mx.MXMatrix(ctx, 0, 64).quantize(empty), w, out)
    mx.MXMatrix(ctx, 0, 64).read(empty)
    ctx.sync()


def test_the_example_with_weights_in_4_bits(ctx):
    """prompts and single tokens through a model whose products run here: every one of them is that of its inputs' and weights' values, in 64
    bits, and the last one's results are the logits that the answers are taken from"""
    from tpu_compiler_amd import kv_example

    class Noted(kv_example.Model4):
        def product(self, x, weights, residual=None):
            y = super().product(x, weights, residual)
            xv, wv = O.values(*O.quantized(x), weights.cols), O.values(weights.codes.numpy(), weights.scales.numpy(), weights.cols)
            want, size = O.product(xv, wv, None, None if residual is None else residual.astype(np.float64))
            assert (np.abs(y - want) <= O.bound(want, size, weights.cols, "f32")).all()
            self.last = y
            calls.append(x.shape)
            return y

    calls = []
    model, rng = Noted(ctx), np.random.default_rng(4)
    prompts = [rng.integers(0, 512, n) for n in (9, 70, 1)]
    answers, steps, _ = kv_example.generate(ctx, model, prompts, 4, 8, page_tokens=32, pages_on_gpu=True)
    assert [len(a) for a in answers] == [4, 4, 4] and calls[0] == (80, 512) and calls[-1] == (3, 512) and len(calls) == 4 * 7
    assert np.array_equal(steps[-1], model.last) and [a[-1] for a in answers] == model.last.argmax(-1).tolist()
    model.close()


def test_torch_tensors_and_streams():
    """in a process of its own, with torch imported first"""
    import os
    import subprocess
    import sys
    run = subprocess.run([sys.executable, "-u", os.path.join(os.path.dirname(os.path.abspath(__file__)), "mx_torch.py")], stdout=subprocess.PIPE,
                         stderr=subprocess.STDOUT, text=True, timeout=110)
    assert run.returncode == 0 and "fine" in run.stdout, run.stdout[-2000:]
