"""A language model's key/value cache held in 4 or 8 bits (tpuhip_kv_*): rows are quantised as they are written, read back, and attended
to from where they lie.  Every call goes to the HIP library; nothing here computes.

Arrays are device memory: `DeviceArray` below, or anything that has torch's data_ptr(), shape, stride() and dtype.  A context works on
a stream of its own; whoever makes arrays on another one passes that stream (`Context(stream=...)`) or waits in between."""
import ctypes as C

import numpy as np

from . import capi

TYPES = {"bf16": 0, "f16": 1, "f32": 2}
_SIZES = {"bf16": 2, "f16": 2, "f32": 4, "i32": 4}
_NAMES = {"bfloat16": "bf16", "float16": "f16", "float32": "f32", "int32": "i32"}


class DeviceArray:
    """A dense array in device memory: "bf16" (numpy holds it as uint16), "f16", "f32" or "i32"."""

    def __init__(self, ctx, shape, dtype):
        self.ctx, self.shape, self.dtype = ctx, tuple(int(n) for n in shape), dtype
        self.size = int(np.prod(self.shape, dtype=np.int64))
        self.nbytes = self.size * _SIZES[dtype]
        self.ptr = ctx.malloc(self.nbytes)

    @classmethod
    def of(cls, ctx, values, dtype):
        """the values, rounded to the type (bf16: of what float32 holds of them)"""
        if dtype == "i32" and np.size(values) and not (-2 ** 31 <= np.min(values) and np.max(values) < 2 ** 31):
            _refuse("values: no ints of 32 bits")
        a = cls(ctx, np.shape(values), dtype)
        if dtype == "bf16":
            bits = np.ascontiguousarray(values, np.float32).view(np.uint32).astype(np.uint64)
            nan = (bits & 0x7FFFFFFF) > 0x7F800000
            host = np.where(nan, 0x7FC0, bits + 0x7FFF + (bits >> 16 & 1) >> 16).astype(np.uint16)
        else:
            host = np.ascontiguousarray(values, {"f16": np.float16, "f32": np.float32, "i32": np.int32}[dtype])
        if a.nbytes:
            ctx.upload(a.ptr, host)
        return a

    def numpy(self):
        """its values: float32 of bf16"""
        host = self.ctx.download(self.ptr, self.shape, {"bf16": np.uint16, "f16": np.float16, "f32": np.float32, "i32": np.int32}[self.dtype])
        return (host.astype(np.uint32) << 16).view(np.float32) if self.dtype == "bf16" else host

    def data_ptr(self):
        return self.ptr

    def stride(self):
        s = [1]
        for n in self.shape[:0:-1]:
            s.append(s[-1] * n)
        return tuple(s[::-1])

    def free(self):
        if self.ptr:
            self.ctx.free(self.ptr)
            self.ptr = None


def _refuse(message):
    raise capi.TpuHipError(1, message)


def _int(n, what):
    """a number for a C int, which would take the low 32 bits of any"""
    n = int(n)
    if not -2 ** 31 <= n < 2 ** 31:
        _refuse("%s: %d is no int of 32 bits" % (what, n))
    return n


def _type(x, what, allowed):
    name = str(x.dtype).replace("torch.", "")
    name = _NAMES.get(name, name)
    if name not in allowed:
        _refuse("%s: of type %s, not %s" % (what, " or ".join(allowed), name))
    return name


def _device(x, what, ctx):
    d = getattr(x, "device", None)      # torch's
    if d is not None and (d.type != "cuda" or (d.index or 0) != ctx.device):
        _refuse("%s: on %s, the context works on device %d" % (what, d, ctx.device))
    own = getattr(x, "ctx", None)       # a DeviceArray's
    if own is not None and own.device != ctx.device:
        _refuse("%s: on device %d, the context works on device %d" % (what, own.device, ctx.device))


def _rows3(x, what, ctx, heads, dim):
    """an array [rows, heads, dim] whose numbers lie next to each other: its strides"""
    _device(x, what, ctx)
    if len(x.shape) != 3 or x.shape[1] != heads or x.shape[2] != dim:
        _refuse("%s: [rows, %d, %d] are wanted, not %s" % (what, heads, dim, tuple(x.shape)))
    st = x.stride()
    if dim > 1 and st[2] != 1:
        _refuse("%s: the numbers of a head lie %d apart" % (what, st[2]))
    return int(st[0]), int(st[1])


def _ints(x, what, ctx, shape):
    _device(x, what, ctx)
    _type(x, what, ("i32",))
    if tuple(x.shape) != shape or (shape[-1] > 1 and x.stride()[-1] != 1):
        _refuse("%s: %s int32 in a row are wanted, not %s" % (what, list(shape), tuple(x.shape)))
    return x.data_ptr()


class _Call:
    """A checked call, to be made any number of times on the same arrays (it keeps them alive) while these, the cache and its context are
    there."""

    def __init__(self, cache, fn, args, keep):
        self._cache, self._ctx, self._fn, self._args, self._keep = cache, cache.ctx, fn, args, keep
        self._arrays = [x for x in keep if isinstance(x, DeviceArray)]
        self._check()

    def _check(self):
        if not self._cache.h or not self._ctx.h:
            _refuse("the %s is closed" % ("context" if not self._ctx.h else "cache"))
        for x in self._arrays:
            if not x.ptr:
                _refuse("an array of the call has been freed")

    def __call__(self):
        self._check()
        if rc := self._fn(self._ctx.h, self._cache.h, *self._args):
            self._ctx._ck(rc)


class KVCache:
    """Pages of `page_tokens` tokens of `kv_heads` heads of `head_dim` numbers, keys and values, in `bits` bits.  Token t of a sequence lies
    in slot page * page_tokens + t % page_tokens of the sequence's page number t // page_tokens; which page that is, is the caller's to say."""

    def __init__(self, ctx, pages, kv_heads, head_dim, bits=4, page_tokens=64):
        self.h = C.c_void_p()
        self.ctx, self.pages, self.kv_heads, self.head_dim = ctx, _int(pages, "pages"), _int(kv_heads, "kv_heads"), _int(head_dim, "head_dim")
        self.bits, self.page_tokens = _int(bits, "bits"), _int(page_tokens, "page_tokens")
        d = capi.KVDesc(self.pages, self.page_tokens, self.kv_heads, self.head_dim, self.bits)
        ctx._ck(ctx.lib.tpuhip_kv_cache_create(ctx.h, C.byref(d), C.byref(self.h)))
        self._made_by = ctx                  # closes this cache before it ends
        ctx.caches.add(self)
        self.nbytes = int(ctx.lib.tpuhip_kv_cache_bytes(C.byref(d)))

    def close(self):
        if self.h:
            self._made_by._ck(self._made_by.lib.tpuhip_kv_cache_destroy(self._made_by.h, self.h))
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:       # its context's stream is being recorded, or the process ends
            self._made_by.unfreed.append(self)

    def _rows(self, fn, slots, k, v):
        tokens = _int(k.shape[0], "tokens")
        ks, vs = _rows3(k, "k", self.ctx, self.kv_heads, self.head_dim), _rows3(v, "v", self.ctx, self.kv_heads, self.head_dim)
        dtype = _type(k, "k", tuple(TYPES))
        if _type(v, "v", tuple(TYPES)) != dtype or v.shape[0] != tokens:
            _refuse("k and v: of one type and length")
        at = _ints(slots, "slots", self.ctx, (tokens,))
        d = capi.KVRows(tokens, TYPES[dtype], k.data_ptr(), v.data_ptr(), *ks, *vs)
        return _Call(self, fn, (d, at), (k, v, slots))

    def plan_write(self, k, v, slots):
        """a call that quantises rows k, v [tokens, kv_heads, head_dim] into slots [tokens] (int32; -1: passed over; a slot twice for the same
        row only)"""
        return self._rows(self.ctx.lib.tpuhip_kv_write, slots, k, v)

    def plan_read(self, slots, k, v):
        """a call that reads the rows in slots back into k, v (zeros for a slot of -1)"""
        return self._rows(self.ctx.lib.tpuhip_kv_read, slots, k, v)

    def plan_attention(self, q, out, q_starts, kv_lens, page_table, max_q=None, max_kv=None, scale=None, window=0, sinks=0):
        """A call in which queries attend to the cache.  q, out: [queries, heads, head_dim], the sequences' one after the other; q_starts
        [sequences + 1], kv_lens [sequences] (the queries' own tokens among them), page_table [sequences, pages]: int32.  out is no part of q.
        A query sees the tokens up to its own, with a window the last `window` of them and the first `sinks` of the sequence.  max_q, max_kv: no
        sequence has more queries or tokens (the fewer, the better the work is split).  scale: 1 / sqrt(head_dim)."""
        heads, total = int(q.shape[1]) if len(q.shape) == 3 else 0, int(q.shape[0])
        qs, outs = _rows3(q, "q", self.ctx, heads, self.head_dim), _rows3(out, "out", self.ctx, heads, self.head_dim)
        dtype = _type(q, "q", ("bf16", "f16"))
        if _type(out, "out", ("bf16", "f16")) != dtype or out.shape[0] != total:
            _refuse("q and out: of one type and length")
        n, most = (int(page_table.shape[0]), int(page_table.shape[1])) if len(page_table.shape) == 2 else (0, 0)
        args = [_ints(q_starts, "q_starts", self.ctx, (n + 1,)), _ints(kv_lens, "kv_lens", self.ctx, (n,)),
                _ints(page_table, "page_table", self.ctx, (n, most))]
        max_kv = min(most * self.page_tokens, 1 << 30) if max_kv is None else int(max_kv)   # a sequence has no more
        if max_kv > most * self.page_tokens:      # the library sees the distance of the table's rows only, which may be parts of longer ones
            _refuse("max_kv: %d tokens in %d pages of %d" % (max_kv, most, self.page_tokens))
        d = capi.KVAttentionDesc(_int(n, "sequences"), _int(heads, "heads"), TYPES[dtype], _int(total, "queries"),
                                 _int(total if max_q is None else max_q, "max_q"), _int(max_kv, "max_kv"), _int(window, "window"), _int(sinks, "sinks"),
                                 _int(page_table.stride()[0] if n > 1 else most, "page_table: distance of rows"),
                                 self.head_dim ** -0.5 if scale is None else float(scale), *qs, *outs)
        return _Call(self, self.ctx.lib.tpuhip_kv_attention, (d, q.data_ptr(), out.data_ptr(), *args),
                     (q, out, q_starts, kv_lens, page_table))

    def write(self, k, v, slots):
        self.plan_write(k, v, slots)()

    def read(self, slots, k, v):
        self.plan_read(slots, k, v)()

    def attention(self, q, out, q_starts, kv_lens, page_table, **how):
        self.plan_attention(q, out, q_starts, kv_lens, page_table, **how)()
