"""Products whose result lies where the call still reads: which are refused.  Stand-ins for torch's tensors, whose views share memory, and for the
library, so no device is needed."""
import itertools
from types import SimpleNamespace

import pytest

from test_kv_calls import Array, context
from tpu_compiler_amd import capi, mx
from tpu_compiler_amd.kv_cache import DeviceArray

SIZES = {"bf16": 2, "f16": 2, "f32": 4, "u8": 1}


class Tensor(Array):
    """a view of memory: from byte `at` on"""
    device = SimpleNamespace(type="cuda", index=0)

    def __init__(self, at, shape, dtype, stride=None):
        super().__init__(shape, dtype, stride)
        self.ptr = at


def matrix(ctx, rows, cols, codes=1 << 30, scales=1 << 31):
    blocks = -(-cols // 32)
    return mx.MXMatrix(ctx, rows, cols, Tensor(codes, (rows, blocks * 16), "u8"), Tensor(scales, (rows, blocks), "u8"))


def refuses(f):
    with pytest.raises(capi.TpuHipError, match="place"):
        f()


def product(ctx, x, out, w=None, **more):
    w = w or matrix(ctx, out.shape[1], x.cols if isinstance(x, mx.MXMatrix) else x.shape[1])
    mx.plan_product(ctx, x, w, out, **more)()


def test_views_of_the_rows():
    ctx, x = context(), Tensor(0x10000, (6, 64), "bf16")
    refuses(lambda: product(ctx, x, Tensor(0x10000, (6, 64), "bf16")))                    # x itself, in another view
    refuses(lambda: product(ctx, x, Tensor(0x10000, (6, 64), "bf16"), residual=x))
    refuses(lambda: product(ctx, x, Tensor(0x10000 + 6 * 128 - 2, (6, 40), "bf16")))      # the last number
    refuses(lambda: product(ctx, x, Tensor(0x10000 - 6 * 80 + 2, (6, 40), "bf16")))       # the first
    refuses(lambda: product(ctx, x, Tensor(0x10000 - 4500, (6, 40), "f32", (400, 1))))    # the fourth of rows that are far apart
    assert "tpuhip_mx_linear" not in ctx.lib.names()
    product(ctx, x, Tensor(0x10000 + 6 * 128, (6, 40), "bf16"))                           # behind it
    product(ctx, x, Tensor(0x10000 - 6 * 80, (6, 40), "bf16"))                            # before it


def test_columns_of_one_array():
    """results beside the rows that they are made of, as fused layers hold them"""
    ctx, row = context(), 200
    for rows in (1, 2, 5000):
        x = Tensor(0x10000, (rows, 64), "bf16", (row, 1))
        product(ctx, x, Tensor(0x10000 + 128, (rows, 136), "bf16", (row, 1)))
        product(ctx, x, Tensor(0x10000 + 200, (rows, 64), "bf16", (row, 1)))
        refuses(lambda: product(ctx, x, Tensor(0x10000 + 126, (rows, 64), "bf16", (row, 1))))
        if rows > 1:
            refuses(lambda: product(ctx, x, Tensor(0x10000 + 274, (rows, 64), "bf16", (row, 1))))   # up to the next row's second number
            refuses(lambda: product(ctx, x, Tensor(0x10000 - 2 * row + 126, (rows, 64), "bf16", (row, 1))))
            product(ctx, x, Tensor(0x10000 + 2 * row * rows, (rows, 64), "bf16", (row, 1)))


def test_the_place_of_a_residual_is_its_own_or_none():
    ctx, x = context(), Tensor(0x90000, (6, 64), "f16")
    out = Tensor(0x10000, (6, 40), "f16", (50, 1))
    product(ctx, x, out, residual=out)
    product(ctx, x, out, residual=Tensor(0x10000, (6, 40), "f16", (50, 1)))               # another view of the same
    product(ctx, x, out, residual=Tensor(0x20000, (6, 40), "f16"))
    product(ctx, x, out, residual=Tensor(0x20000, (6, 40), "f16", (0, 1)))                # one row for all
    refuses(lambda: product(ctx, x, out, residual=Tensor(0x10000, (6, 40), "f16", (40, 1))))   # rows elsewhere
    refuses(lambda: product(ctx, x, out, residual=Tensor(0x10000, (6, 40), "f16", (0, 1))))
    refuses(lambda: product(ctx, x, out, residual=Tensor(0x10002, (6, 40), "f16", (50, 1))))
    one = Tensor(0x10000, (1, 40), "f16", (50, 1))
    product(ctx, Tensor(0x90000, (1, 64), "f16"), one, residual=Tensor(0x10000, (1, 40), "f16", (40, 1)))


def test_weights_biases_and_rows_in_4_bits():
    ctx, x, out = context(), Tensor(0x90000, (6, 64), "f32"), Tensor(0x10000, (6, 40), "f32")
    end = 0x10000 + 6 * 160
    refuses(lambda: product(ctx, x, out, bias=Tensor(end - 4, (40,), "f32")))
    product(ctx, x, out, bias=Tensor(end, (40,), "f32"))
    refuses(lambda: product(ctx, x, out, w=matrix(ctx, 40, 64, codes=end - 16)))
    refuses(lambda: product(ctx, x, out, w=matrix(ctx, 40, 64, scales=end - 1)))
    product(ctx, x, out, w=matrix(ctx, 40, 64, codes=end, scales=0x10000 - 80))
    w = matrix(ctx, 40, 64, codes=0x50000, scales=0x60000)
    refuses(lambda: product(ctx, matrix(ctx, 6, 64, codes=0x10000), out, w=w))
    refuses(lambda: product(ctx, matrix(ctx, 6, 64, scales=end - 1), out, w=w))
    product(ctx, matrix(ctx, 6, 64), out, w=w)


def test_rows_that_are_quantised_or_read_in_their_own_place():
    ctx = context()
    m = matrix(ctx, 6, 64, codes=0x10000, scales=0x20000)
    for plan in (m.plan_quantize, m.plan_read):
        refuses(lambda: plan(Tensor(0x10000 - 6 * 256 + 4, (6, 64), "f32")))
        refuses(lambda: plan(Tensor(0x20000 + 8, (6, 64), "bf16")))
        plan(Tensor(0x10000 - 6 * 256, (6, 64), "f32"))()


def test_memory_of_one_s_own_is_told_by_the_object():
    ctx = context()
    a, b = DeviceArray(ctx, (6, 64), "f32"), DeviceArray(ctx, (6, 64), "f32")             # the stand-in's are all at one address
    product(ctx, a, b, residual=b)
    refuses(lambda: product(ctx, a, a))


def test_rows_meet_as_their_bytes_do():
    """against the bytes themselves"""
    spans = [(start, rows, stride, width) for start in (0, 3, 8, 21) for rows in (1, 2, 5) for stride in (0, 4, 7, 12) for width in (1, 4)
             if stride >= width or stride == 0]
    bytes_of = {s: {s[0] + i * s[2] + k for i in range(s[1]) for k in range(s[3])} for s in spans}
    for a, b in itertools.product(spans, spans):
        assert mx._meet(a, b) == bool(bytes_of[a] & bytes_of[b]), (a, b)
