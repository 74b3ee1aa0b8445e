"""The Python side of the key/value cache: what calls are made with, and which are refused.  A stand-in for the library notes its calls, so
no device is needed."""
import ctypes as C
import gc

import pytest

from tpu_compiler_amd import capi
from tpu_compiler_amd.kv_cache import KVCache


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name,) + args)
            if name == "tpuhip_kv_cache_create":
                args[2]._obj.value = 0x1000
            if name == "tpuhip_malloc":
                args[2]._obj.value = 0x2000
            return 0
        return call

    def names(self):
        return [c[0] for c in self.calls]


def context():
    ctx = capi.Context.__new__(capi.Context)
    ctx._begin(Library(), 0, C.c_void_p(0x10))
    return ctx


class Array:
    """device memory of some shape"""
    ptr = 0x5000

    def __init__(self, shape, dtype, stride=None):
        self.shape, self.dtype, self._stride = shape, dtype, stride

    def data_ptr(self):
        return self.ptr

    def stride(self):
        if self._stride:
            return self._stride
        s = [1]
        for n in self.shape[:0:-1]:
            s.append(s[-1] * n)
        return tuple(s[::-1])


def plans(cache, rows=3, seqs=2, pages=4):
    k, v, q, out = (Array((rows, h, 64), "bf16") for h in (2, 2, 4, 4))
    slots = Array((rows,), "i32")
    return [cache.plan_write(k, v, slots), cache.plan_read(slots, k, v),
            cache.plan_attention(q, out, Array((seqs + 1,), "i32"), Array((seqs,), "i32"), Array((seqs, pages), "i32"))]


def test_a_plan_passes_the_handles_of_its_cache_and_context():
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 32)
    for plan, name in zip(plans(cache), ("tpuhip_kv_write", "tpuhip_kv_read", "tpuhip_kv_attention")):
        for _ in range(2):
            plan()
            call = ctx.lib.calls[-1]
            assert call[0] == name and call[1].value == 0x10 and call[2].value == 0x1000


@pytest.mark.parametrize("what", ["cache", "context"])
def test_a_plan_whose_cache_or_context_is_closed_refuses(what):
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 32)
    made = plans(cache)
    (cache if what == "cache" else ctx).close()
    before = len(ctx.lib.calls)
    for plan in made:
        with pytest.raises(capi.TpuHipError, match="closed"):
            plan()
    assert len(ctx.lib.calls) == before


def test_a_context_that_closes_frees_its_caches_first():
    ctx = context()
    kept = KVCache(ctx, 8, 2, 64, 4, 32)
    gone = KVCache(ctx, 8, 2, 64, 4, 32)
    gone.close()
    ctx.close()
    assert ctx.lib.names().count("tpuhip_kv_cache_destroy") == 2
    assert ctx.lib.names()[-1] == "tpuhip_ctx_destroy" and ctx.lib.names()[-2] == "tpuhip_kv_cache_destroy"
    kept.close()
    assert ctx.lib.names()[-1] == "tpuhip_ctx_destroy"


def test_a_plan_whose_array_is_freed_refuses():
    from tpu_compiler_amd.kv_cache import DeviceArray
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 32)
    k, v, slots = DeviceArray(ctx, (3, 2, 64), "bf16"), DeviceArray(ctx, (3, 2, 64), "bf16"), DeviceArray(ctx, (3,), "i32")
    write = cache.plan_write(k, v, slots)
    write()
    v.free()
    before = len(ctx.lib.calls)
    with pytest.raises(capi.TpuHipError, match="freed"):
        write()
    with pytest.raises(capi.TpuHipError, match="freed"):
        cache.plan_write(k, v, slots)
    assert len(ctx.lib.calls) == before


def attend(cache, table, **how):
    q, out = (Array((2, 4, 64), "bf16") for _ in range(2))
    return cache.plan_attention(q, out, Array((table.shape[0] + 1,), "i32"), Array((table.shape[0],), "i32"), table, **how)


def test_no_more_tokens_than_a_page_table_lists():
    """rows of a table may be parts of longer ones: what lies behind them is none of the table's, and past the last row no memory at all"""
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 32)
    for table in (Array((2, 4), "i32"), Array((2, 4), "i32", (40, 1)), Array((1, 4), "i32", (40, 1))):
        attend(cache, table, max_kv=128)()
        call = ctx.lib.calls[-1]
        assert call[3].max_kv == 128 and call[3].table_stride == (table.stride()[0] if table.shape[0] > 1 else 4)
        with pytest.raises(capi.TpuHipError, match="4 pages"):
            attend(cache, table, max_kv=129)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 4, -2 ** 31 - 1, 2 ** 40])
def test_numbers_that_an_int_does_not_hold_are_refused(n):
    """and not taken for what is left of them in 32 bits"""
    ctx = context()
    for place in range(5):
        sizes = [8, 2, 64, 4, 32]
        sizes[place] = n
        with pytest.raises(capi.TpuHipError, match="int"):
            KVCache(ctx, *sizes)
    cache = KVCache(ctx, 8, 2, 64, 4, 32)
    for name in ("max_q", "max_kv", "window", "sinks"):
        with pytest.raises(capi.TpuHipError):
            attend(cache, Array((2, 4), "i32"), **{name: n})
    with pytest.raises(capi.TpuHipError, match="int"):
        attend(cache, Array((2, 4), "i32", (n, 1)))
    if n > 0:
        with pytest.raises(capi.TpuHipError, match="int"):
            cache.plan_write(Array((n, 2, 64), "bf16"), Array((n, 2, 64), "bf16"), Array((n,), "i32"))


def test_a_table_of_more_pages_than_a_sequence_has():
    """by default a call looks at no more than 2^30 tokens, the most there may be"""
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 1 << 20)
    attend(cache, Array((2, 5000), "i32"))()
    assert ctx.lib.calls[-1][3].max_kv == 1 << 30


@pytest.mark.parametrize("values", [[2 ** 31], [-2 ** 31 - 1], [2 ** 32 + 3]])
def test_integers_that_do_not_fit_are_not_uploaded(values):
    from tpu_compiler_amd.kv_cache import DeviceArray
    ctx = context()
    with pytest.raises(capi.TpuHipError, match="int"):
        DeviceArray.of(ctx, values, "i32")
    DeviceArray.of(ctx, [2 ** 31 - 1, -2 ** 31], "i32")


def test_torch_tensors_of_other_devices_types_and_orders():
    import torch
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 32)

    class Placed:
        """a tensor that says it lies on a device"""
        def __init__(self, x, device):
            self.x, self.device = x, torch.device(device)

        def __getattr__(self, name):
            return getattr(self.x, name)

    k, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3, dtype=torch.int32)
    here = lambda x: Placed(x, "cuda:0")
    cache.plan_write(here(k), here(k), here(slots))()
    assert ctx.lib.calls[-1][3].dtype == 0 and ctx.lib.calls[-1][3].k == k.data_ptr() and ctx.lib.calls[-1][4] == slots.data_ptr()
    part = torch.zeros(3, 7, 70)[:, 2:4, 3:67]
    cache.plan_write(here(part), here(part), here(slots))()
    d = ctx.lib.calls[-1][3]
    assert d.dtype == 2 and (d.k_token_stride, d.k_head_stride) == (490, 70) and d.k == part.data_ptr()
    for bad, says in ((k, "on cpu"), (Placed(k, "cuda:1"), "on cuda:1"), (here(k.double()), "float64"), (here(k[:, :1]), "are wanted"),
                      (here(torch.zeros(3, 2, 128, dtype=torch.bfloat16)[:, :, ::2]), "lie 2 apart")):
        with pytest.raises(capi.TpuHipError, match=says):
            cache.plan_write(bad, here(k), here(slots))
    with pytest.raises(capi.TpuHipError, match="int64"):
        cache.plan_write(here(k), here(k), here(slots.long()))


@pytest.mark.parametrize("prompts", [[], [[1, 2], []]])
def test_the_example_refuses_prompts_without_a_token(prompts):
    """there is nothing to continue, and the logits of another sequence would be taken for its own"""
    from tpu_compiler_amd import kv_example
    ctx = context()
    with pytest.raises(ValueError, match="token"):
        kv_example.generate(ctx, kv_example.Model(), prompts, 3)
    assert not ctx.lib.calls


def test_the_example_gives_out_pages_until_there_are_no_more():
    from tpu_compiler_amd import kv_example
    ctx = context()
    s = kv_example.Sequences(ctx, 1, 8, 2, 64, 4, pages=3, page_tokens=32)
    s.begin([40, 20])
    with pytest.raises(ValueError, match="pages"):
        s.begin([30, 0])
    assert s.lens == [40, 20] and len(s.pages[0]) == 2
    s.begin([24, 12])                            # what fits is taken all the same
    assert s.lens == [64, 32]


def test_a_cache_that_could_not_be_freed_can_be_closed_again():
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 32)
    status = [2]
    ctx.lib.tpuhip_kv_cache_destroy = lambda *a: status[0]
    ctx.lib.tpuhip_last_error = lambda: b"a stream is being captured"
    with pytest.raises(capi.TpuHipError, match="captured"):
        cache.close()
    status[0] = 0
    assert cache.h
    cache.close()
    assert not cache.h


def test_a_cache_that_is_collected_while_it_cannot_be_freed_is_freed_with_its_context():
    ctx = context()
    cache = KVCache(ctx, 8, 2, 64, 4, 32)
    freed = []
    ctx.lib.tpuhip_last_error = lambda: b"a stream is being captured"
    ctx.lib.tpuhip_kv_cache_destroy = lambda *a: 1
    del cache
    gc.collect()
    ctx.lib.tpuhip_kv_cache_destroy = lambda c, h: freed.append(h.value) or 0
    ctx.close()
    assert freed == [0x1000]
