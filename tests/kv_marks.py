"""Inputs of attention to a quantised cache that show a token left out, counted twice or read in another's place, at any length.

  counting  all scores are alike, and each token adds the largest code to one channel: a result is a number of tokens over a number of tokens
  finding   keys are patterns, and a query is that of one token, which then has all the weight: the result is its values.  Tokens just
            outside of what a query sees have the pattern of one that it looks for"""
import numpy as np

import kv_bounds
import kv_oracle as O

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}     # half a unit of a result


def channels(n, dim):
    """of every other token the next one, of those between by where they lie: a part of a sequence that is left out takes its own"""
    t = np.arange(n)
    return np.where(t % 2 == 0, (7 * t + t // dim) % dim, t // -(-n // dim))


def counting(kv_lens, kv_heads, dim, bits):
    """values of each sequence: one channel of a row is the largest code, the others zero, exactly"""
    out = []
    for n in kv_lens:
        v = np.zeros((n, kv_heads, dim), np.float32)
        v[np.arange(n), :, channels(n, dim)] = 2 ** bits - 1
        out.append(v)
    return out


def counted(kv_lens, q_lens, dim, bits, window=0, sinks=0, seen=kv_bounds.seen):
    """-> [rows, dim]: what every head of a query gets"""
    out = np.zeros((sum(q_lens), dim))
    row = 0
    for n, q in zip(kv_lens, q_lens):
        c = channels(n, dim)
        for i in range(q):
            t = seen(n - q + i, n, window, sinks)
            if len(t):
                out[row] = np.bincount(c[t], minlength=dim) * (2 ** bits - 1) / len(t)
            row += 1
    return out


def counting_limit(want, dtype):
    """a weight is 1 and codes are whole numbers, which 32 bits hold: the quotient's two roundings and the result's are left"""
    return (UNIT[dtype] + 2.0 ** -21) * want


def finding(rng, kv_lens, q_lens, heads, kv_heads, dim, bits, window=0, sinks=0):
    """-> q [rows, heads, dim], k, v of each sequence, the scale"""
    top, q, ks, vs = 2 ** bits - 1, [], [], []
    for n, count in zip(kv_lens, q_lens):
        on = rng.random((n, kv_heads, dim)) < 0.5
        on[:, :, 0], on[:, :, 1] = False, True                   # a row's offset and step are 0 and 1
        look = np.zeros((count, heads), np.int64)
        for i in range(count):
            t = kv_bounds.seen(n - count + i, n, window, sinks)
            if not len(t):
                continue
            edges = [t[0], t[-1], t[min(len(t) - 1, sinks)], t[max(0, min(len(t), sinks) - 1)], t[-1] // 32 * 32, t[len(t) // 2]]
            edges += [x for x in (1, 15, 16, 31, 32, 63, 64, len(t) - 33, len(t) - 2) if 0 <= x < len(t)]
            edges = [x for x in edges if x in t] + list(rng.choice(t, heads))
            look[i] = [edges[(h + i) % len(edges)] if i % 2 == 0 else rng.choice(t) for h in range(heads)]
        patterns = on.copy()
        if count:
            p = n - 1
            for j, hidden in enumerate({p - window, sinks} if window else ()):
                if sinks <= hidden <= p - window:
                    for g in range(kv_heads):
                        on[hidden, g] = patterns[look[-1, g * heads // kv_heads + j % (heads // kv_heads)], g]
        of_head = np.arange(heads) * kv_heads // heads
        q.append(np.where(patterns[look, of_head], 1.0, -1.0).astype(np.float32))
        ks.append(np.where(on, float(top), 0.0).astype(np.float32))
        vs.append(O.rounded(rng.standard_normal((n, kv_heads, dim)), "bf16"))
    return np.concatenate(q), ks, vs, 1.0 if bits == 4 else 1 / 16


def found(q, k, v, bits, q_lens, kv_lens, scale, window=0, sinks=0, seen=kv_bounds.seen, held=O.values):
    heads, out, row = q.shape[1], np.zeros(q.shape), 0
    for kk, vv, count, n in zip(k, v, q_lens, kv_lens):
        group, vv = heads // kk.shape[1], held(vv, bits) if n else vv
        sees = np.zeros((count, n), bool)
        for i in range(count):
            sees[i, seen(n - count + i, n, window, sinks)] = True
        for g in range(kk.shape[1] if n else 0):
            at = np.s_[row:row + count, g * group:(g + 1) * group]
            x = np.where(sees[:, None], q[at] @ kk[:, g].T * np.float32(scale), -np.inf)     # whole numbers: exact
            w = np.exp((x - np.maximum(x.max(-1, keepdims=True), -1e30)).astype(np.float64)) * sees[:, None]
            out[at] = w @ vv[:, g] / np.maximum(w.sum(-1, keepdims=True), 1e-300)
        row += count
    return out


def finding_limit(want, dtype):
    """Weights are 1 (or of two or three tokens alike): 2^-13 off at most, as scores of up to 3000 in units of log 2 are rounded, a sixth of a
    float16's rounding, which makes 1 of them again; the sum of weights is not rounded so.  Values are 6 at most, and so are their codes'
    and their offset's parts."""
    return UNIT[dtype] * np.abs(want) + 6 * 2.0 ** -12
