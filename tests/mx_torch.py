"""Microscaled numbers and a batch's pages on torch tensors; run by test_gpu_mx.py, with torch imported first."""
import os
import sys

import torch

sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))]
import mx_oracle as O  # noqa: E402
from tpu_compiler_amd import capi, mx  # noqa: E402
from tpu_compiler_amd.kv_cache import KVCache, KVPages  # noqa: E402


def values(x):
    return torch.from_numpy(O.values(*O.quantized(x.float().cpu().numpy()), x.shape[1])).to(x.device)


def layer(ctx, dtype, rows, width, cols):
    """what torch makes just before goes through a quantised layer, and torch works on the result just after; parts of larger tensors throughout"""
    weights = torch.randn(cols, width + 3, device="cuda")[:, 3:] / width ** 0.5
    w = mx.MXMatrix(ctx, cols, width, codes=torch.zeros(cols, -(-width // 32) * 16, dtype=torch.uint8, device="cuda"),
                    scales=torch.zeros(cols, -(-width // 32), dtype=torch.uint8, device="cuda"))
    w.quantize(weights)
    bias = torch.randn(cols, device="cuda")
    for _ in range(3):
        x = (torch.randn(rows, 2 * width, device="cuda") @ torch.eye(2 * width, device="cuda")).to(dtype)[:, width:]
        both = torch.full((rows, 2, cols), 7.0, dtype=dtype, device="cuda")
        residual = torch.randn(rows, cols, device="cuda").to(dtype)
        mx.product(ctx, x, w, both[:, 0], bias=bias, residual=residual)
        doubled = both * 2
        xv, wv = values(x), values(weights)
        want, size = xv @ wv.T + bias.double() + residual.double(), xv.abs() @ wv.abs().T + bias.abs() + residual.abs().double()
        name = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}[dtype]
        bound = (-(-width // 32) + 18) * 2.0 ** -23 * size + O.HALF_STEP[name] * want.abs() + O.SMALLEST[name] + 2.0 ** -100
        assert (both[:, 1] == 7).all()
        assert ((doubled[:, 0].double() / 2 - want).abs() <= bound).all(), (dtype, rows, width, cols)


def pages(ctx):
    """a batch's step: pages, slots, rows into a cache and back"""
    n, page = 5, 32
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    p = KVPages(ctx, 40, n, 8, page, lens=i32(0, 0, 0, 0, 0), table=torch.full((n, 8), -1, dtype=torch.int32, device="cuda"),
                free=torch.randperm(40, device="cuda").to(torch.int32), n_free=i32(40))
    cache = KVCache(ctx, 40, 2, 64, 8, page)
    new = i32(10, 0, 33, 64, 1) + (torch.ones(n, device="cuda") * 2).to(torch.int32)
    starts, slots = torch.zeros(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(130, dtype=torch.int32, device="cuda")
    p.grow(new, starts, slots)
    assert torch.equal(starts, torch.cat([i32(0), torch.cumsum(new, 0).to(torch.int32)])) and torch.equal(p.lens, new)
    total = int(starts[-1])
    assert (slots[total:] == -1).all() and len(set(slots[:total].tolist())) == total
    k, v = (torch.randn(130, 2, 64, device="cuda") for _ in range(2))
    cache.write(k, v, slots)
    back = [torch.empty_like(k) for _ in range(2)]
    cache.read(slots, *back)
    for a, b in zip(back, (k, v)):
        step = (b.amax(-1, keepdim=True) - b.amin(-1, keepdim=True)) / 255
        assert ((a - b)[:total].abs() <= step[:total]).all() and not a[total:].any()
    p.trim(i32(0, 0, 0, 0, 0))
    assert int(p.n_free) == 40 and (p.table == -1).all()
    torch.cuda.current_stream().synchronize()
    cache.close()


def main():
    torch.manual_seed(0)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            ctx = capi.Context(stream=stream.cuda_stream)
            for dtype in (torch.bfloat16, torch.float16, torch.float32):
                for rows, width, cols in ((1, 512, 100), (5, 70, 33), (40, 300, 129), (300, 1000, 700)):
                    layer(ctx, dtype, rows, width, cols)
            pages(ctx)
            ctx.close()
    print("fine")


main()
