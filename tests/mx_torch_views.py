"""Products of torch's tensors that are views of one memory; run by test_gpu_mx_views.py, with torch imported first."""
import os
import sys

import torch

sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))]
import mx_oracle as O  # noqa: E402
from tpu_compiler_amd import capi, mx  # noqa: E402


def refuses(f):
    try:
        f()
    except capi.TpuHipError as e:
        assert "place" in str(e), e
    else:
        raise AssertionError("not refused")


def main():
    torch.manual_seed(0)
    ctx = capi.Context(stream=torch.cuda.current_stream().cuda_stream)
    for rows in (3, 70, 300):
        k, n = 96, 80
        codes = [torch.zeros(n, k // 32 * b, dtype=torch.uint8, device="cuda") for b in (16, 1)]
        weights = torch.randn(n, k, device="cuda")
        w = mx.MXMatrix(ctx, n, k, *codes).quantize(weights)
        square = mx.MXMatrix(ctx, k, k).quantize(torch.randn(k, k, device="cuda"))
        buffer = torch.randn(rows, k + n + 7, device="cuda")
        x, y, more = buffer[:, :k], buffer[:, k:k + n], buffer[:, k:k + n]       # rows and results beside each other, y in two views
        value = lambda v: torch.from_numpy(O.values(*O.quantized(v.cpu().numpy()), k))
        want, size = O.product(value(x).numpy(), value(weights).numpy(), None, y.double().cpu().numpy())
        before = buffer.clone()
        mx.product(ctx, x, w, y, residual=more)
        assert (abs(y.double().cpu().numpy() - want) <= O.bound(want, size, k, "f32")).all()
        assert torch.equal(buffer[:, :k], before[:, :k]) and torch.equal(buffer[:, k + n:], before[:, k + n:])
        dense, before = x.contiguous(), buffer.clone()
        refuses(lambda: mx.product(ctx, dense, square, dense.view(rows, k)))
        refuses(lambda: mx.product(ctx, x, w, buffer[:, k - 1:k - 1 + n]))
        refuses(lambda: mx.product(ctx, x, w, y, residual=buffer[:, k + 1:k + 1 + n]))
        refuses(lambda: mx.product(ctx, x, w, y, bias=buffer.view(-1)[k:k + n]))
        assert torch.equal(buffer, before)
    torch.cuda.synchronize()
    ctx.close()
    print("fine")


main()
