"""The oracles of microscaled numbers and of a batch's pages against the plain forms that performance is measured against, on the CPU; run by
test_mx_oracle.py."""
import importlib.util
import os

import numpy as np
import torch

import mx_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("more_operators", os.path.join(ROOT, "perf", "more_operators.py"))
plain = importlib.util.module_from_spec(spec)
spec.loader.exec_module(plain)
plain.DEVICE = "cpu"


def rows(rng):
    for cols in (1, 31, 32, 33, 700, 2050):
        x = (rng.standard_normal((9, cols)) * 2.0 ** rng.integers(-120, 121, (9, 1)) * 2.0 ** rng.integers(-6, 7, (1, cols))).astype(np.float32)
        x[0] = 0
        x[1] = 2.0 ** -140
        x[2] = (rng.integers(-32, 33, cols) / 4).astype(np.float32)        # ties
        x[3] = np.float32(3e38) * rng.choice([-1, 1, 0.3, 0], cols).astype(np.float32)
        yield x


def quantised(rng):
    for x in rows(rng):
        codes, scales = O.quantized(x)
        c, s = plain._quantised(torch.from_numpy(x))
        assert np.array_equal(codes, c.numpy()) and np.array_equal(scales, s.numpy())
        with np.errstate(over="ignore"):
            assert np.array_equal(O.values(codes, scales, x.shape[1]).astype(np.float32), plain._values(c, s, x.shape[1]).numpy())
        for dtype, torch_dtype in (("bf16", torch.bfloat16), ("f16", torch.float16)):
            assert np.array_equal(O.rounded(x, dtype), torch.from_numpy(x).to(torch_dtype).float().numpy())


def products(rng):
    for n, cols in ((1, 1), (5, 70), (9, 2050)):
        x, w, bias, more = (rng.standard_normal(s) for s in ((n, cols), (n + 3, cols), (n + 3,), (n, n + 3)))
        y, size = O.product(x, w, bias, more)
        a, b, c, d = (torch.from_numpy(v) for v in (x, w, bias, more))
        want = (a[:, None] * b).sum(-1) + c + d
        sizes = (a[:, None] * b).abs().sum(-1) + c.abs() + d.abs()
        assert np.abs(y - want.numpy()).max() <= 2 * cols * 2.0 ** -53 * size.max() and np.allclose(size, sizes.numpy(), rtol=1e-12)


def pages(rng):
    refused = 0
    for n, count, most, page in ((1, 9, 9, 32), (40, 120, 6, 32), (7, 200, 50, 96)):
        o = O.Pages(count, n, most, page)
        s = dict(case=dict(page=page), lens=torch.zeros(n, dtype=torch.int32), table=torch.full((n, most), -1, dtype=torch.int32),
                 free=torch.arange(count - 1, -1, -1, dtype=torch.int32), n_free=torch.tensor([count], dtype=torch.int32),
                 q_starts=torch.zeros(n + 1, dtype=torch.int32), refused=torch.zeros(1, dtype=torch.int32))
        for step in range(60):
            new = rng.integers(0, rng.choice([2, 10, 3 * page]), n)
            s["slots"] = torch.zeros(int(rng.choice([max(new.sum(), 1), new.sum() + 9, new.sum() // 2 + 1])), dtype=torch.int32)
            plain._grow(s, torch.from_numpy(new.astype(np.int32)))
            starts, slots, short = o.grow(new.tolist(), s["slots"].numel())
            refused += short
            assert s["q_starts"].tolist() == starts and s["slots"].tolist() == [int(v) for v in slots] and int(s["refused"]) == short
            if step % 3 == 2:
                keep = rng.integers(0, np.array(o.lens) + 3)
                plain._trim(s, torch.from_numpy(keep.astype(np.int32)))
                o.trim(keep.tolist())
            assert s["lens"].tolist() == o.lens and np.array_equal(s["table"].numpy(), o.table())
            assert int(s["n_free"]) == len(o.free) and s["free"][:len(o.free)].tolist() == o.free
    assert refused


for check in (quantised, products, pages):
    check(np.random.default_rng(0))
print("fine")
