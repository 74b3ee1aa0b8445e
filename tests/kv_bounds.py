"""How far attention to a quantised cache may be from its formula, row by row, from the terms of that row alone."""
import numpy as np

import kv_oracle as O


def seen(p, length, window, sinks):
    """the tokens that a query at position p sees"""
    t = np.arange(max(0, min(p + 1, length)))
    return t[(t > p - window) | (t < sinks)] if window else t


def attention(q, k, v, bits, q_lens, kv_lens, scale, dtype, window=0, sinks=0):
    """q [rows, H, D]; k, v: a list of [tokens, KH, D] of each sequence before they are quantised -> (want, limit) [rows, H, D], 64 bits.

    With a token's keys m + s c, its score is x = scale (s q.c + m sum(q)), of terms that come to T = scale (s |q|.c + |m| sum|q|), and its
    weight p.  Roundings, u = 2^-24:
      a score     at most D + 8 of 32 bits, each of T or less, and one of the largest score, which is taken off: the weight is that much off,
                  and its share of the result with it: p ((D + 8) u T + 4 u max|x| + 8 u) (|V| + |out|), 8 u the exponential and products
      a weight    times its step to float16, 2^-11 of its term: p s c, or for a float16 result p s |c - L / 2|; one that is small beside the
                  largest step S loses at most 2^-30 S c (that is held as 2^5 or more, where float16 ends at 2^-25)
      the sums    32 bits, no more than n / 16 + 64 additions one after the other, of the terms p |m| and p s c
      the result  half a unit of 8 or 11 bits: bfloat16 numbers from 1 on lie 2^-7 apart, float16 numbers 2^-10"""
    heads, dim = q.shape[1:]
    want, limit = np.zeros(q.shape), np.zeros(q.shape)
    u, unit = 2.0 ** -24, {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    row = 0
    for kk, vv, n, length in zip(k, v, q_lens, kv_lens):
        (kc, ks, km), (vc, vs, vm) = ((O.quantise(x, bits) if len(x) else (np.zeros(x.shape), *[np.zeros(x.shape[:2] + (1,))] * 2)) for x in (kk, vv))
        for i in range(n):
            t = seen(length - n + i, length, window, sinks)
            for h in range(heads if len(t) else 0):
                g = h * kk.shape[1] // heads
                qq = q[row, h].astype(np.float64)
                x = scale * ((km + ks * kc)[t, g] @ qq)
                terms = abs(scale) * (ks[t, g, 0] * (kc[t, g] @ np.abs(qq)) + np.abs(km[t, g, 0]) * np.abs(qq).sum())
                w = np.exp(x - x.max())
                w /= w.sum()
                codes, offsets = vs[t, g] * vc[t, g], vm[t, g]
                out = w @ (offsets + codes)
                off = w * ((dim + 8) * u * terms + 4 * u * np.abs(x).max() + 8 * u)
                part, c = w @ codes, vc[t, g]
                rounded = w @ (vs[t, g] * np.abs(c - (2 ** bits - 1) / 2)) if dtype == "f16" else part
                want[row, h] = out
                limit[row, h] = unit * np.abs(out) + off @ (np.abs(offsets + codes) + np.abs(out)) + 2.0 ** -11 * rounded + \
                    2.0 ** -30 * vs[t, g].max() * c.sum(0) * w.max() + (len(t) / 16 + 64) * u * (w @ np.abs(offsets) + part) + 2.0 ** -126
                if dtype == "f16":
                    limit[row, h] += 2.0 ** -25
            row += 1
    return want, limit
