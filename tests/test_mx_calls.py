"""The Python side of microscaled numbers and of a batch's pages: what calls are made with, and which are refused; their oracles against each
other.  A stand-in for the library notes its calls, so no device is needed."""
import gc
from fractions import Fraction

import numpy as np
import pytest

import mx_oracle as O
from test_kv_calls import Array, context
from tpu_compiler_amd import capi, mx
from tpu_compiler_amd.kv_cache import DeviceArray, KVPages


def matrix(ctx, rows, cols, c_stride=None, s_stride=None):
    blocks = -(-cols // 32)
    return mx.MXMatrix(ctx, rows, cols, Array((rows, blocks * 16), "u8", c_stride), Array((rows, blocks), "u8", s_stride))


def refuses(f, says):
    with pytest.raises(capi.TpuHipError, match=says):
        f()


def test_quantising_and_reading_pass_what_they_are_given():
    ctx = context()
    m = matrix(ctx, 5, 70, (96, 1), (9, 1))
    for plan, name in ((m.plan_quantize(Array((5, 70), "f16", (100, 1))), "tpuhip_mx_quantize"), (m.plan_read(Array((5, 70), "f32")), "tpuhip_mx_read")):
        for _ in range(2):
            plan()
        call = ctx.lib.calls[-1]
        assert call[0] == name and call[1].value == 0x10 and call[3] == Array.ptr
        d = call[2]
        assert (d.rows, d.cols, d.codes_stride, d.scales_stride) == (5, 70, 96, 9)
        assert call[4:] == ((1, 100) if name.endswith("quantize") else (2, 70))


def test_products_pass_what_they_are_given():
    ctx = context()
    w, out = matrix(ctx, 40, 70), Array((6, 40), "bf16", (50, 1))
    mx.plan_product(ctx, matrix(ctx, 6, 70), w, out)()
    name, h, d, x, m, y = ctx.lib.calls[-1]
    assert name == "tpuhip_mx_product" and (x.rows, x.cols, m.rows, m.cols, y) == (6, 70, 40, 70, Array.ptr)
    assert (d.dtype, d.y_stride, d.bias, d.residual) == (0, 50, None, None)
    mx.plan_product(ctx, Array((6, 70), "f32", (80, 1)), w, out, bias=Array((40,), "f32"), residual=Array((6, 40), "bf16"))()
    name, h, d, x, dtype, stride, room, m, y = ctx.lib.calls[-1]
    assert name == "tpuhip_mx_linear" and (x, dtype, stride, y) == (Array.ptr, 2, 80, Array.ptr)
    assert (room.rows, room.cols) == (6, 70) and room.codes_stride % 128 == 0 and room.codes_stride >= 48 and room.scales_stride >= 3
    assert room.scales == room.codes + 6 * room.codes_stride
    assert (d.bias, d.residual, d.residual_stride) == (Array.ptr, Array.ptr, 40)


@pytest.mark.parametrize("x,out,more,says", [
    (Array((6, 71), "f32"), Array((6, 40), "bf16"), {}, "71 columns"),
    (Array((6,), "f32"), Array((6, 40), "bf16"), {}, "are wanted"),
    (Array((6, 70), "i32"), Array((6, 40), "bf16"), {}, "type"),
    (Array((6, 70), "f32", (70, 2)), Array((6, 40), "bf16"), {}, "apart"),
    (Array((6, 70), "f32"), Array((5, 40), "bf16"), {}, "are wanted"),
    (Array((6, 70), "f32"), Array((6, 41), "bf16"), {}, "are wanted"),
    (Array((6, 70), "f32"), Array((6, 40), "u8"), {}, "type"),
    (Array((6, 70), "f32"), Array((6, 40), "f16"), dict(residual=Array((6, 40), "bf16")), "one type"),
    (Array((6, 70), "f32"), Array((6, 40), "f16"), dict(residual=Array((6, 4), "f16")), "are wanted"),
    (Array((6, 70), "f32"), Array((6, 40), "f16"), dict(bias=Array((40,), "f16")), "type"),
    (Array((6, 70), "f32"), Array((6, 40), "f16"), dict(bias=Array((39,), "f32")), "bias"),
    (Array((6, 70), "f32"), Array((6, 40), "f16"), dict(bias=Array((40,), "f32", (2,))), "bias"),
])
def test_products_that_are_refused(x, out, more, says):
    ctx = context()
    refuses(lambda: mx.plan_product(ctx, x, matrix(ctx, 40, 70), out, **more), says)
    assert not [c for c in ctx.lib.calls if "mx" in c[0]]


def test_a_product_in_the_place_of_its_rows_is_refused():
    ctx, x = context(), Array((6, 70), "f32")
    refuses(lambda: mx.plan_product(ctx, x, matrix(ctx, 70, 70), x), "place")
    mx.plan_product(ctx, Array((6, 70), "f32"), matrix(ctx, 70, 70), x, residual=x)()


def test_matrices_that_are_refused():
    ctx = context()
    codes, scales = Array((4, 48), "u8"), Array((4, 3), "u8")
    refuses(lambda: mx.MXMatrix(ctx, 4, 0), "columns")
    refuses(lambda: mx.MXMatrix(ctx, -1, 3), "rows")
    refuses(lambda: mx.MXMatrix(ctx, 2 ** 31, 3), "int")
    refuses(lambda: mx.MXMatrix(ctx, 4, 70, codes), "both")
    refuses(lambda: mx.MXMatrix(ctx, 4, 70, Array((4, 47), "u8"), scales), "are wanted")
    refuses(lambda: mx.MXMatrix(ctx, 4, 70, codes, Array((4, 4), "u8")), "are wanted")
    refuses(lambda: mx.MXMatrix(ctx, 4, 70, Array((4, 48), "i32"), scales), "type")
    refuses(lambda: matrix(ctx, 4, 70).plan_quantize(Array((4, 71), "f32")), "are wanted")
    refuses(lambda: mx.plan_product(ctx, Array((6, 70), "f32"), Array((40, 70), "f32"), Array((6, 40), "f32")), "no MXMatrix")
    other = context()
    other.device = 1
    refuses(lambda: mx.plan_product(ctx, matrix(ctx, 6, 70), matrix(other, 40, 70), Array((6, 40), "f32")), "device 1")


def test_the_memory_that_x_is_quantised_in_goes_from_plan_to_plan_and_ends_with_the_context():
    ctx = context()
    w, plan = matrix(ctx, 40, 70), lambda rows: mx.plan_product(ctx, Array((rows, 70), "f32"), w, Array((rows, 40), "f32"))
    a, b = plan(6), plan(6)
    made = lambda: ctx.lib.names().count("tpuhip_malloc")
    assert made() == 2                                       # two plans at a time may not share it: one of them may be recorded
    del a
    gc.collect()
    c = plan(5)
    assert made() == 2
    d = plan(5)
    assert made() == 3
    del b
    gc.collect()
    e = plan(100)                                            # larger than what is there
    assert made() == 4
    ctx.close()
    assert ctx.lib.names().count("tpuhip_free") == 4 and ctx.lib.names()[-1] == "tpuhip_ctx_destroy"
    for p in (c, d, e):
        refuses(p, "closed")


def test_a_plan_whose_matrix_is_freed_refuses():
    ctx = context()
    w = mx.MXMatrix(ctx, 40, 70)
    plans = [mx.plan_product(ctx, Array((6, 70), "f32"), w, Array((6, 40), "f32")), w.plan_read(Array((40, 70), "f32"))]
    w.free()
    for p in plans:
        refuses(p, "freed")


def test_pages_pass_what_they_are_given():
    ctx = context()
    p = KVPages(ctx, 50, 3, 7, 32)
    assert ctx.lib.names()[-1] == "tpuhip_kv_pages_clear"
    p.grow(Array((3,), "i32"), Array((4,), "i32"), Array((90,), "i32"), Array((1,), "i32"))
    name, h, d, new, capacity, starts, slots, refused = ctx.lib.calls[-1]
    assert name == "tpuhip_kv_pages_grow" and capacity == 90 and refused == Array.ptr
    assert (d.n_seq, d.pages, d.page_tokens, d.max_pages, d.table_stride) == (3, 50, 32, 7, 7)
    p.grow(Array((3,), "i32"), Array((4,), "i32"), Array((90,), "i32"))
    assert ctx.lib.calls[-1][-1] is None
    p.trim(Array((3,), "i32"))
    assert ctx.lib.calls[-1][0] == "tpuhip_kv_pages_trim"
    arrays = dict(lens=Array((3,), "i32"), table=Array((3, 7), "i32", (20, 1)), free=Array((50,), "i32"), n_free=Array((1,), "i32"))
    before = len(ctx.lib.calls)
    q = KVPages(ctx, 50, 3, 7, 32, **arrays)
    assert len(ctx.lib.calls) == before                      # their state goes on
    q.trim(Array((3,), "i32"))
    assert ctx.lib.calls[-1][2].table_stride == 20
    for name, wrong in (("lens", (4,)), ("table", (3, 6)), ("free", (49,)), ("n_free", (2,))):
        refuses(lambda: KVPages(ctx, 50, 3, 7, 32, **dict(arrays, **{name: Array(wrong, "i32")})), name)
        refuses(lambda: KVPages(ctx, 50, 3, 7, 32, **dict(arrays, **{name: Array(arrays[name].shape, "f32")})), "type")
        refuses(lambda: KVPages(ctx, 50, 3, 7, 32, **dict(arrays, **{name: None})), "all of them")
    for sizes in ((0, 3, 7), (50, 0, 7), (50, 3, 0), (2 ** 31, 3, 7)):
        refuses(lambda: KVPages(ctx, *sizes), "pages|sequences|int")
    for new, starts, slots in (((4,), (4,), (9,)), ((3,), (3,), (9,)), ((3,), (4,), (3, 3))):
        refuses(lambda: p.plan_grow(Array(new, "i32"), Array(starts, "i32"), Array(slots, "i32")), "wanted")
    refuses(lambda: p.plan_trim(Array((2,), "i32")), "keep")


def test_bytes_that_do_not_fit_are_not_uploaded():
    ctx = context()
    for bad in ([256], [-1]):
        refuses(lambda: DeviceArray.of(ctx, bad, "u8"), "bytes")


def test_the_example_takes_back_what_a_refused_step_got():
    """the stand-in's memory is what was uploaded: a count of refused sequences says how the step ends"""
    from tpu_compiler_amd import kv_example
    ctx = context()
    s = kv_example.SequencesOnGpu(ctx, 1, 8, 2, 64, 4, 3, 2, page_tokens=32)
    answer = [0]
    ctx.download = lambda ptr, shape, dtype: np.array(answer, dtype)
    s.begin([40, 20])
    assert s.lens == [40, 20] and s.step["max_kv"] == 40
    s.end()
    answer[0] = 1
    with pytest.raises(ValueError, match="pages"):
        s.begin([60, 1])
    assert s.lens == [40, 20] and "tpuhip_kv_pages_trim" in ctx.lib.names()


def test_the_oracle_quantises_by_the_definition():
    """against exact fractions, over every kind of number"""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((30, 64)) * 2.0 ** rng.integers(-60, 60, (30, 1))).astype(np.float32)
    x[0, :9] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5]
    x[1] = 0
    x[2, 32:] = 2.0 ** -140
    codes, scales = O.quantized(x)
    table = [Fraction(float(v)) for v in O.VALUES[:8]]
    for row in range(30):
        for block in range(2):
            v = [Fraction(float(u)) for u in x[row, block * 32:block * 32 + 32]]
            top = max(abs(u) for u in v)
            e = -127
            while e < 127 and Fraction(2) ** (e + 3) <= top:
                e += 1
            assert scales[row, block] == e + 127
            for i, u in enumerate(v):
                c = int(codes[row, block * 16 + i // 2] >> 4 * (i % 2) & 15)
                size = abs(u) / Fraction(2) ** e
                best = min(abs(size - t) for t in table)
                near = [k for k, t in enumerate(table) if abs(size - t) == best]
                assert c & 7 == (near[0] if len(near) == 1 else next(k for k in near if k % 2 == 0))
                assert c >> 3 == int(np.signbit(x[row, block * 32 + i]))


def test_a_mistake_is_out_of_the_products_bound():
    """a block left out, a code read for its neighbour, a scale off by one: more than what rounding does, for results of every type"""
    rng = np.random.default_rng(1)
    cols = 2048
    x, w = (O.values(*O.quantized(rng.standard_normal((n, cols))), cols) for n in (6, 9))
    want, size = O.product(x, w)
    less = w.copy()
    less[:, 640:672] = 0
    swapped = x.copy()
    swapped[:, [100, 101]] = swapped[:, [101, 100]]
    scaled = w.copy()
    scaled[:, 32:64] *= 2
    for dtype in ("f32", "f16", "bf16"):
        for a, b in ((x, less), (x, scaled)) + (((swapped, w),) if dtype != "bf16" else ()):
            off = np.abs(O.product(a, b)[0] - want) > O.bound(want, size, cols, dtype)
            assert off.mean() > 0.5
