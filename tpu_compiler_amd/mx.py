"""Rows of microscaled 4-bit floating point numbers (tpuhip_mx_*; the OCP format MXFP4): quantised, read back, multiplied.  Every call goes to the
HIP library; nothing here computes.

Arrays are device memory as kv_cache takes it: DeviceArray, or anything that has torch's data_ptr(), shape, stride() and dtype."""
from . import capi
from .kv_cache import _SIZES, TYPES, DeviceArray, _device, _int, _Plan, _refuse, _type

BLOCK = 32


def _rows2(x, what, ctx, rows, cols):
    """an array [rows, cols] whose columns lie next to each other: the distance of its rows"""
    _device(x, what, ctx)
    if len(x.shape) != 2 or x.shape[0] != rows or x.shape[1] != cols:
        _refuse("%s: [%d, %d] are wanted, not %s" % (what, rows, cols, tuple(x.shape)))
    st = x.stride()
    if cols > 1 and st[1] != 1:
        _refuse("%s: the numbers of a row lie %d apart" % (what, st[1]))
    return int(st[0]) if rows > 1 else cols


def _span(x, dtype, rows, cols, stride):
    """an array and where its rows lie: (address, rows, their distance, bytes of one); an address of None if nothing else can lie there.  Tensors of torch's may
    be views of one memory; a DeviceArray's is its own, and what else there is does not say."""
    size = _SIZES[dtype]
    return x, (x.data_ptr() if rows and getattr(x, "device", None) is not None else None, rows, stride * size, cols * size)


def _meet(a, b):
    """whether rows share bytes"""
    (at_a, rows_a, step_a, width_a), (at_b, rows_b, step_b, width_b) = a, b
    if at_a + (rows_a - 1) * step_a + width_a <= at_b or at_b + (rows_b - 1) * step_b + width_b <= at_a:
        return False
    once = (s if s[1] > 1 and s[2] else (s[0], 1, 1, s[3]) for s in (a, b))
    (at_a, rows_a, step_a, width_a), (at_b, rows_b, step_b, width_b) = sorted(once, key=lambda s: s[1])
    if step_a == step_b:                             # then row i of one and row j of the other lie as any others with the same i - j do
        first = at_a - at_b
        k = min((width_b - 1 - first) // step_a, rows_a - 1)
        return k > -rows_b and first + k * step_a > -width_a
    # the last row of b that begins before a's row ends
    return any(at_b + min((at + width_a - 1 - at_b) // step_b, rows_b - 1) * step_b + width_b > at
               for at in range(at_a, at_a + (rows_a - 1) * step_a + 1, step_a) if at + width_a > at_b)


def _apart(x, y, what):
    """refuses the span x where it shares memory with y"""
    if x[0] is y[0] or (x[1][0] is not None and y[1][0] is not None and _meet(x[1], y[1])):
        _refuse(what)


class MXMatrix:
    """[rows, cols] numbers in 4 bits: codes [rows, 16 a block] and scales [rows, blocks], uint8, a block 32 columns.  Made here (with what memory
    holds, until something is quantised into it) or the caller's, as a file of weights has them."""

    def __init__(self, ctx, rows, cols, codes=None, scales=None):
        self.ctx, self.rows, self.cols = ctx, _int(rows, "rows"), _int(cols, "cols")
        if self.rows < 0 or self.cols < 1:
            _refuse("a matrix of %d rows, %d columns" % (self.rows, self.cols))
        if (codes is None) != (scales is None):
            _refuse("codes and scales: both of them or none")
        self.blocks = -(-self.cols // BLOCK)
        if codes is None:
            codes, scales = DeviceArray(ctx, (self.rows, 16 * self.blocks), "u8"), DeviceArray(ctx, (self.rows, self.blocks), "u8")
        self.codes, self.scales = codes, scales
        _type(codes, "codes", ("u8",)), _type(scales, "scales", ("u8",))
        strides = [_rows2(codes, "codes", ctx, self.rows, 16 * self.blocks), _rows2(scales, "scales", ctx, self.rows, self.blocks)]
        self._spans = [_span(x, "u8", self.rows, width, stride) for x, width, stride in zip((codes, scales), (16 * self.blocks, self.blocks), strides)]
        self._d = capi.MXMatrixDesc(self.rows, self.cols, codes.data_ptr(), scales.data_ptr(), *strides)

    @property
    def nbytes(self):
        return self.rows * self.blocks * 17

    def _plan(self, fn, x, what):
        dtype, stride = _type(x, what, tuple(TYPES)), _rows2(x, what, self.ctx, self.rows, self.cols)
        for own in self._spans:
            _apart(_span(x, dtype, self.rows, self.cols, stride), own, "%s in the place of the matrix" % what)
        return _Plan(self.ctx, fn, (self._d, x.data_ptr(), TYPES[dtype], stride), (self.codes, self.scales, x))

    def plan_quantize(self, x):
        """a call that quantises x [rows, cols], bf16, f16 or f32, into this matrix"""
        return self._plan(self.ctx.lib.tpuhip_mx_quantize, x, "x")

    def plan_read(self, out):
        """a call that writes what the matrix stands for to out"""
        return self._plan(self.ctx.lib.tpuhip_mx_read, out, "out")

    def quantize(self, x):
        self.plan_quantize(x)()
        return self

    def read(self, out):
        self.plan_read(out)()

    def free(self):
        """frees its DeviceArrays; other arrays are their owners'"""
        for a in (self.codes, self.scales):
            if isinstance(a, DeviceArray):
                a.free()


class _Room:
    """Memory in which a call quantises x.  It is its context's, and goes from a plan that nobody holds to the next one of its size: calls on one
    context follow each other, and freeing it would wait for them, which nothing may do while they are recorded.  Sizes are powers of two, so that
    products of any lengths come to hold four times what the largest need at most, for as many of them as there are at a time; a plan takes no larger
    one than its own, as it may stay for good."""
    SMALLEST = 4096

    def __init__(self, ctx, nbytes):
        self.array, self.taken = DeviceArray(ctx, (nbytes,), "u8"), True

    @classmethod
    def take(cls, ctx, nbytes):
        size = max(cls.SMALLEST, 1 << (nbytes - 1).bit_length())
        for r in ctx.rooms:
            if not r.taken and r.array.nbytes == size:
                r.taken = True
                return r
        r = cls(ctx, size)
        ctx.rooms.append(r)
        return r

    def free(self):
        self.array.free()


class _Linear(_Plan):
    """a product that quantises x"""

    def __init__(self, ctx, room, *args):
        self._room = room
        super().__init__(ctx, *args)

    def __del__(self):
        self._room.taken = False


def plan_product(ctx, x, w, out, bias=None, residual=None):
    """A call that computes out = x w^T (+ bias) (+ residual).  w: an MXMatrix [columns of out, k]; x: one too, [rows of out, k], or an array of
    bf16, f16 or f32, which the call quantises (in memory that the plan keeps).  out, residual (may be out): bf16, f16 or f32, [rows, columns]; bias:
    f32, [columns].  out shares memory with nothing else that the call reads (checked of torch's tensors, which may be views of one memory).  A plan
    that quantises is made before a recording, not in it: it may need memory."""
    if not isinstance(w, MXMatrix):
        _refuse("w: no MXMatrix")
    if not isinstance(x, MXMatrix) and len(x.shape) != 2:
        _refuse("x: [rows, %d] are wanted, not %s" % (w.cols, tuple(x.shape)))
    rows, k = (x.rows, x.cols) if isinstance(x, MXMatrix) else (_int(x.shape[0], "rows"), int(x.shape[1]))
    if k != w.cols:
        _refuse("x has %d columns, w %d" % (k, w.cols))
    for m in (x, w):
        if isinstance(m, MXMatrix) and m.ctx.device != ctx.device:
            _refuse("a matrix lies on device %d, the context works on device %d" % (m.ctx.device, ctx.device))
    dtype = _type(out, "out", tuple(TYPES))
    if not isinstance(x, MXMatrix):
        stride, x_type = _rows2(x, "x", ctx, rows, k), _type(x, "x", tuple(TYPES))
    d = capi.MXProductDesc(TYPES[dtype], _rows2(out, "out", ctx, rows, w.rows), 0, None, None)
    here = _span(out, dtype, rows, w.rows, d.y_stride)
    for part in x._spans if isinstance(x, MXMatrix) else (_span(x, x_type, rows, k, stride),):
        _apart(here, part, "out in the place of x")
    for part in w._spans:
        _apart(here, part, "out in the place of w")
    if bias is not None:
        _device(bias, "bias", ctx)
        _type(bias, "bias", ("f32",))
        if tuple(bias.shape) != (w.rows,) or (w.rows > 1 and bias.stride()[0] != 1):
            _refuse("bias: %d numbers in a row are wanted, not %s" % (w.rows, tuple(bias.shape)))
        _apart(here, _span(bias, "f32", 1, w.rows, 0), "out in the place of the bias")
        d.bias = bias.data_ptr()
    if residual is not None:
        if _type(residual, "residual", tuple(TYPES)) != dtype:
            _refuse("out and residual: of one type")
        d.residual, d.residual_stride = residual.data_ptr(), _rows2(residual, "residual", ctx, rows, w.rows)
        if d.residual != out.data_ptr() or d.residual_stride != d.y_stride:
            _apart(here, _span(residual, dtype, rows, w.rows, d.residual_stride), "out neither in the residual's place nor apart from it")
    keep = (w.codes, w.scales, out, bias, residual)
    if isinstance(x, MXMatrix):
        return _Plan(ctx, ctx.lib.tpuhip_mx_product, (d, x._d, w._d, out.data_ptr()), keep + (x.codes, x.scales))
    codes, scales = -(-w.blocks // 8) * 128, -(-w.blocks // 16) * 16      # rows that begin at lines of the caches
    room = _Room.take(ctx, rows * (codes + scales))
    at = room.array.data_ptr()
    m = capi.MXMatrixDesc(rows, k, at, at + rows * codes, codes, scales)
    return _Linear(ctx, room, ctx.lib.tpuhip_mx_linear, (d, x.data_ptr(), TYPES[x_type], stride, m, w._d, out.data_ptr()), keep + (x, room.array))


def product(ctx, x, w, out, bias=None, residual=None):
    plan_product(ctx, x, w, out, bias, residual)()
