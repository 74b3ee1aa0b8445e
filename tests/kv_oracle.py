"""The key/value cache's operators from their formulas, in 64 bits (numpy).  Bfloat16 numbers are held as float32 here."""
import numpy as np


def bf16(x):
    """rounded to bfloat16"""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + (b >> 16 & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def rounded(x, dtype):
    """what a type holds of 64-bit numbers (through float32 for bf16: the callers' numbers have at most 24 bits)"""
    with np.errstate(over="ignore"):
        return {"bf16": lambda v: bf16(np.asarray(v, np.float32)), "f16": lambda v: np.asarray(v, np.float16).astype(np.float32),
                "f32": lambda v: np.asarray(v, np.float32)}[dtype](x)


def _grid(v):
    """the distance of bfloat16 numbers of v's size"""
    return 2.0 ** (np.frexp(np.maximum(np.abs(v), 2.0 ** -126))[1] - 8.0)


def quantise(x, bits):
    """x [..., D] float32 -> codes, steps, offsets (the last two [..., 1], 64 bits; offset NaN for a row that cannot be held)"""
    top = 2 ** bits - 1
    with np.errstate(all="ignore"):
        wide = np.asarray(x, np.float64)
        fine = np.isfinite(wide).all(-1, keepdims=True)
        wide = np.where(fine, wide, 0.0)
        low = wide.min(-1, keepdims=True)
        m = np.floor(low / _grid(low)) * _grid(low)
        span = wide.max(-1, keepdims=True) - m
        s = np.ceil(span / top / _grid(span / top)) * _grid(span / top)
        s = np.where(s < 2.0 ** -126, 0.0, s)
        fine &= span <= np.finfo(np.float32).max
        c = np.where(s > 0, np.clip(np.rint((wide - m) / np.where(s > 0, s, 1)), 0, top), 0)
    return np.where(fine, c, 0), np.where(fine, s, 0), np.where(fine, m, np.nan)


def values(x, bits):
    c, s, m = quantise(x, bits)
    return m + s * c


def attention(q, k, v, q_lens, kv_lens, scale, window=0, sinks=0):
    """q [rows, H, D]; k, v: a list of [tokens, KH, D] of each sequence, 64 bits -> (out, sum of p |v|) [rows, H, D]"""
    heads, dim = q.shape[1:]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    row = 0
    for kk, vv, n, length in zip(k, v, q_lens, kv_lens):
        for i in range(n):
            p = length - n + i
            t = np.arange(max(0, p + 1))
            if window:
                t = t[(t > p - window) | (t < sinks)]
            if len(t):
                for h in range(heads):
                    g = h * kk.shape[1] // heads
                    with np.errstate(all="ignore"):
                        x = kk[t, g] @ q[row, h].astype(np.float64) * scale
                        w = np.exp(x - x.max())
                        w /= w.sum()
                        out[row, h] = w @ vv[t, g]
                        size[row, h] = w @ np.abs(vv[t, g])
            row += 1
    return out, size


def attention_of_finite(q, k, v, q_lens, kv_lens, scale, window=0, sinks=0):
    """the same where all numbers are finite, a cache head's rows at a time"""
    heads, dim = q.shape[1:]
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    row = 0
    for kk, vv, n, length in zip(k, v, q_lens, kv_lens):
        p, t = length - n + np.arange(n)[:, None], np.arange(length)
        seen = (t <= p) & ((t > p - window) | (t < sinks)) if window else t <= p
        group = heads // kk.shape[1]
        for g in range(kk.shape[1]):
            at = np.s_[row:row + n, g * group:(g + 1) * group]
            x = np.where(seen[:, None], q[at].astype(np.float64) @ kk[:, g].T.astype(np.float64) * scale, -np.inf)
            w = np.exp(x - np.maximum(x.max(-1, keepdims=True, initial=-np.inf), -1e300)) * seen[:, None]
            w /= np.maximum(w.sum(-1, keepdims=True), 1e-300)
            out[at], size[at] = w @ vv[:, g].astype(np.float64), w @ np.abs(vv[:, g]).astype(np.float64)
        row += n
    return out, size
