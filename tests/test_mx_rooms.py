"""The memory in which products quantise their rows: how much of it a context comes to hold.  A stand-in for the library notes its calls, so
no device is needed."""
import gc

import pytest

from test_kv_calls import Array, context
from tpu_compiler_amd import mx


def plan(ctx, w, rows):
    return mx.plan_product(ctx, Array((rows, w.cols), "bf16"), w, Array((rows, w.rows), "bf16"))


def weights(ctx, rows, cols):
    blocks = -(-cols // 32)
    return mx.MXMatrix(ctx, rows, cols, Array((rows, blocks * 16), "u8"), Array((rows, blocks), "u8"))


def held(ctx):
    return sum(a[2] for a in made(ctx))


def made(ctx):
    return [(c[0], c[1], c[2]) for c in ctx.lib.calls if c[0] == "tpuhip_malloc"]


@pytest.fixture
def ctx():
    """its calls of malloc as (name, context, bytes)"""
    c = context()
    inner = c.malloc

    def malloc(nbytes):
        ptr = inner(nbytes)
        c.lib.calls[-1] = ("tpuhip_malloc", c.h, int(nbytes))
        return ptr
    c.malloc = malloc
    return c


def need(w, rows):
    """bytes of codes and scales, as plan_product lays them out"""
    return rows * (-(-w.blocks // 8) * 128 + -(-w.blocks // 16) * 16)


@pytest.mark.parametrize("order", ["rising", "falling", "mixed"])
@pytest.mark.parametrize("alive", [1, 3])
def test_products_of_many_lengths_hold_a_few_rooms(ctx, order, alive):
    """one size of memory for each power of two, as many of each as there were plans at a time: four times what the largest of them need"""
    w = weights(ctx, 64, 8192)
    lengths = {"rising": list(range(1, 2049)), "falling": list(range(2048, 0, -1)), "mixed": [i * 769 % 2048 + 1 for i in range(2048)]}[order]
    plans = []
    for rows in lengths:
        plans = plans[-alive + 1:] if alive > 1 else []
        plans.append(plan(ctx, w, rows))
    gc.collect()
    assert held(ctx) <= alive * 4 * need(w, 2048)
    assert len(made(ctx)) <= alive * 24


def test_a_small_product_that_stays_does_not_keep_a_large_room(ctx):
    """layers prepared one after the other: a prompt goes through each, then the layer's plan for single tokens is kept"""
    w, kept = weights(ctx, 64, 8192), []
    for _ in range(80):
        plan(ctx, w, 4096)
        kept.append(plan(ctx, w, 1))
    gc.collect()
    assert held(ctx) <= 2 * need(w, 4096) + 80 * 2 * max(need(w, 1), 4096)


def test_a_room_is_large_enough_and_one_plan_s_at_a_time(ctx):
    w = weights(ctx, 64, 700)
    plans = [plan(ctx, w, rows) for rows in (1, 2, 5, 16, 17, 40, 41, 300, 300, 1)]
    rooms = [p._room for p in plans]
    assert len(set(map(id, rooms))) == len(rooms)
    assert all(r.array.nbytes >= need(w, p._keep[2].shape[0]) for r, p in zip(rooms, plans))


def test_a_matrix_of_the_caller_s_arrays_has_nothing_to_free(ctx):
    """a tensor of torch's is freed when nobody holds it"""
    weights(ctx, 64, 700).free()
    assert "tpuhip_free" not in ctx.lib.names()
    own = mx.MXMatrix(ctx, 64, 700)
    own.free()
    assert ctx.lib.names().count("tpuhip_free") == 2
