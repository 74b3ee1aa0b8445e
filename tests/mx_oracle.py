"""Microscaled 4-bit numbers and a batch's pages by their definitions, in 64 bits and in plain Python."""
import numpy as np

VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}      # of a rounding, relative
SMALLEST = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24, "f32": 2.0 ** -149}    # numbers of a type


def rounded(x, dtype):
    """what an array of the type holds of the values: float32"""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    if dtype == "f32":
        return x
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + (b >> 16 & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def quantized(x):
    """rows [rows, cols] -> codes [rows, blocks * 16], scales [rows, blocks]"""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    x = np.concatenate([np.asarray(x, np.float64), np.zeros((rows, blocks * 32 - cols))], 1).reshape(rows, blocks, 32)
    top = np.abs(x).max(-1)                      # a NaN stays
    fine = np.isfinite(top)
    e = np.clip(np.frexp(np.where(fine, top, 1))[1] - 1 - 2, -127, None)
    e = np.where(top == 0, -127, e)
    size = np.where(fine[..., None], np.abs(x), 0) * 2.0 ** -e[..., None]
    # the nearest of eight values; of two as near, that of the even code
    far = np.abs(size[..., None] - VALUES[:8])
    near = far.min(-1, keepdims=True)
    at = far == near
    code = np.where(at[..., 0::2].any(-1), at[..., 0::2].argmax(-1) * 2, at.argmax(-1)).astype(np.uint8)
    code = np.where(fine[..., None], code | np.signbit(x).astype(np.uint8) << 3, 0).reshape(rows, -1)
    return (code[:, 0::2] | code[:, 1::2] << 4).astype(np.uint8), np.where(fine, e + 127, 255).astype(np.uint8)


def values(codes, scales, cols):
    rows = codes.shape[0]
    c = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1, 32)
    scale = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (VALUES[c] * scale[..., None]).reshape(rows, -1)[:, :cols]


def product(x, w, bias=None, residual=None):
    """(x w^T + bias + residual, the sum of the terms' sizes) of matrices of values"""
    y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    for more in (bias, residual):
        if more is not None:
            y, size = y + more, size + np.abs(more)
    return y, size


def bound(y, size, cols, dtype):
    """How far a result may be from the sum: a block's 32 products are multiples of a power of two below 2^13 of them, so that their sum is exact;
    blocks, sixteen partial sums, bias and residual are added in 32 bits, each addition off by a unit of what it makes, which is not more than
    `size`, if it truncates; then the rounding to the type."""
    return (-(-cols // 32) + 18) * 2.0 ** -23 * size + HALF_STEP[dtype] * np.abs(y) + SMALLEST[dtype] + 2.0 ** -126 * (cols + 1)


class Pages:
    """a batch's pages, one token after the other"""

    def __init__(self, pages, sequences, max_pages, page):
        self.free, self.lens, self.rows = list(range(pages))[::-1], [0] * sequences, [[] for _ in range(sequences)]
        self.max_pages, self.page = max_pages, page

    def grow(self, new, capacity):
        """-> (starts, slots, refused)"""
        starts, slots, refused, wanted_pages, wanted_tokens, have = [0], [], 0, 0, 0, len(self.free)
        for i, n in enumerate(new):
            n = max(n, 0)
            if self.lens[i] + n <= min(self.max_pages * self.page, 1 << 30):
                need = -(-(self.lens[i] + n) // self.page) - len(self.rows[i])
                wanted_pages += need
                wanted_tokens += n
                if wanted_tokens <= capacity and (need == 0 or wanted_pages <= have):
                    for _ in range(need):
                        self.rows[i].append(self.free.pop())
                    at = np.arange(self.lens[i], self.lens[i] + n)
                    slots += list(np.array(self.rows[i] or [0])[at // self.page] * self.page + at % self.page)
                    self.lens[i] += n
                    n = 0
            refused += n > 0
            starts.append(len(slots))
        return starts, slots + [-1] * (capacity - len(slots)), refused

    def trim(self, keep):
        gone = []
        for i, k in enumerate(keep):
            self.lens[i] = min(self.lens[i], max(k, 0))
            left = -(-self.lens[i] // self.page)
            gone += self.rows[i][left:]
            del self.rows[i][left:]
        self.free += gone[::-1]

    def table(self):
        return np.array([r + [-1] * (self.max_pages - len(r)) for r in self.rows], np.int32)
