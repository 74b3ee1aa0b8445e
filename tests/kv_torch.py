"""The key/value cache on torch tensors; run by test_gpu_kv_edges.py, with torch imported first."""
import os
import sys

import torch

sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__)))]
from tpu_compiler_amd import capi  # noqa: E402
from tpu_compiler_amd.kv_cache import KVCache  # noqa: E402


def held(x, bits):
    """what the cache makes of rows, in 64 bits, on the CPU, where a quotient is rounded as it has to be"""
    top, x, device = 2 ** bits - 1, x.cpu().double(), x.device

    def grid(v):
        return 2.0 ** (torch.frexp(v.abs().clamp(min=2.0 ** -126)).exponent.double() - 8)

    low = x.amin(-1, keepdim=True)
    m = torch.floor(low / grid(low)) * grid(low)
    step = (x.amax(-1, keepdim=True) - m) / top
    s = torch.ceil(step / grid(step)) * grid(step)
    return (m + s * torch.round((x - m) / s.clamp(min=1e-300)).clamp(0, top)).to(device)


def attended(q, k, v, first):
    """q [n, heads, d] at positions first.. of k, v [tokens, kv_heads, d]"""
    group = q.shape[1] // k.shape[1]
    out = torch.empty_like(q, dtype=torch.float64)
    for h in range(q.shape[1]):
        x = q[:, h].double() @ k[:, h // group].T.contiguous() / q.shape[2] ** 0.5
        seen = torch.arange(k.shape[0], device=q.device) <= first + torch.arange(q.shape[0], device=q.device)[:, None]
        out[:, h] = torch.softmax(x.masked_fill(~seen, float("-inf")), -1) @ v[:, h // group]
    return out


def step(ctx, dtype, heads, kv_heads, dim, n, new):
    """a prompt of n tokens and then `new` more, queries, keys and values parts of one tensor that torch computes just before and a result that it
    works on just after"""
    page, bits = 32, 8
    cache = KVCache(ctx, -(-(n + new) // page) + 1, kv_heads, dim, bits, page)
    pages = torch.randperm(cache.pages, device="cuda", dtype=torch.int32)[None, :-1].contiguous()
    weight = torch.randn(dim, (heads + 2 * kv_heads) * dim, device="cuda") / dim ** 0.5
    at, ks, vs = 0, [], []
    for count in (n, new):
        x = torch.randn(count, dim, device="cuda")
        qkv = (x @ weight).to(dtype).view(count, heads + 2 * kv_heads, dim)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
        place = torch.arange(at, at + count, device="cuda")
        slots = (pages[0, place // page] * page + place % page).to(torch.int32)
        cache.write(k, v, slots)
        both = torch.full((count, 2, heads, dim), 7.0, dtype=dtype, device="cuda")
        cache.attention(q, both[:, 0], torch.tensor([0, count], dtype=torch.int32, device="cuda"),
                        torch.tensor([at + count], dtype=torch.int32, device="cuda"), pages)
        doubled = both * 2
        back = [torch.empty(count, kv_heads, dim, dtype=torch.float32, device="cuda") for _ in range(2)]
        cache.read(slots, *back)
        ks.append(held(k, bits)), vs.append(held(v, bits))
        for got, want in zip(back, (ks[-1], vs[-1])):
            assert torch.equal(got, want.float())
        want = attended(q, torch.cat(ks), torch.cat(vs), at)
        assert (both[:, 1] == 7).all()
        # float16 weights, half a unit of the result, of numbers of size one
        assert (doubled[:, 0].double() / 2 - want).abs().max() < 2.0 ** -6 * want.abs().max(), (dtype, heads, dim, n)
        at += count
    torch.cuda.current_stream().synchronize()
    cache.close()


def main():
    torch.manual_seed(0)
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            ctx = capi.Context(stream=stream.cuda_stream)
            for dtype in (torch.bfloat16, torch.float16):
                for heads, kv_heads, dim, n, new in ((8, 2, 64, 100, 1), (6, 6, 80, 33, 5), (4, 1, 128, 700, 1)):
                    step(ctx, dtype, heads, kv_heads, dim, n, new)
            ctx.close()
    print("fine")


main()
