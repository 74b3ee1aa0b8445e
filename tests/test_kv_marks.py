"""The inputs and bounds that attention to the cache is tested with, by oracles with a mistake in them: each has to be out of bounds."""
import numpy as np
import pytest

import kv_bounds
import kv_marks as M
import kv_oracle as O
from test_gpu_kv_marked import CASES

LONG = ([131072], [1], 8, 1, 0, 0)


def without(*what):
    """a mistake in which tokens are seen"""
    def seen(p, length, window, sinks):
        t = kv_bounds.seen(p, length, window, sinks)
        for w in what:
            t = w(t, p, length, window, sinks)
        return t
    return seen


MISTAKES = {
    "the last token": without(lambda t, p, *_: t[t != p]),
    "a token more": lambda p, length, window, sinks: kv_bounds.seen(min(p + 1, length), length + 1, window and window + 1, sinks) % length,
    "the first token": without(lambda t, *_: t[1:]),
    "a unit": without(lambda t, *_: t[(t // 32) != t[len(t) // 2] // 32] if len(t) else t),
    "a token twice": without(lambda t, *_: np.append(t, t[len(t) // 3]) if len(t) else t),
    "a window one too large": lambda p, length, window, sinks: kv_bounds.seen(p, length, window + 1, sinks),
    "a window one too small": lambda p, length, window, sinks: kv_bounds.seen(p, length, window - 1, sinks),
    "a first token too many": lambda p, length, window, sinks: kv_bounds.seen(p, length, window, sinks + 1),
    "a first token too few": lambda p, length, window, sinks: kv_bounds.seen(p, length, window, max(0, sinks - 1)),
    "a split": without(lambda t, *_: t[(t < t[len(t) // 2]) | (t >= t[len(t) // 2] + len(t) // 16)] if len(t) > 64 else t[:0]),
}


@pytest.mark.parametrize("bits,dim,dtype", [(4, 128, "f16"), (8, 80, "bf16")])
@pytest.mark.parametrize("mistake", MISTAKES)
@pytest.mark.parametrize("case", CASES + [LONG])
def test_a_wrong_set_of_tokens_is_out_of_bounds(case, mistake, bits, dim, dtype):
    kv_lens, q_lens, heads, kv_heads, window, sinks = case
    if ("window" in mistake and not window) or (mistake == "a window one too small" and window == 1):
        return
    if case == LONG:
        dim, dtype = 256, "f16"
    n, q = kv_lens[0], q_lens[0]
    if dtype == "bf16" and n > 60 * dim:
        return                                                   # 8 bits do not tell a token among more
    if n == 1 and mistake in ("a token more", "a token twice"):
        return                                                   # the only one there is
    if "first token too" in mistake and (not window or not sinks <= n - window - 1 or ("few" in mistake and not sinks)):
        return
    q = min(q, 3)                                                # the last of the first sequence's queries
    want = M.counted([n], [q], dim, bits, window, sinks)[-1]
    wrong = M.counted([n], [q], dim, bits, window, sinks, seen=MISTAKES[mistake])[-1]
    assert (np.abs(wrong - want) > 2 * M.counting_limit(want, dtype)).any()   # as far from what a kernel may give


@pytest.mark.parametrize("bits,dim,dtype", [(4, 128, "f16"), (8, 64, "f16"), (4, 72, "bf16")])
@pytest.mark.parametrize("case", [c for c in CASES if sum(c[1]) <= 40 and max(c[0]) <= 9000])
def test_mistakes_in_what_is_found_are_out_of_bounds(case, bits, dim, dtype):
    kv_lens, q_lens, heads, kv_heads, window, sinks = case
    rng = np.random.default_rng(sum(kv_lens))
    q, k, v, scale = M.finding(rng, kv_lens, q_lens, heads, kv_heads, dim, bits, window, sinks)
    v = [O.values(x, bits) for x in v]
    as_held = lambda x, b: x
    want = M.found(q, k, v, bits, q_lens, kv_lens, scale, window, sinks, held=as_held)
    limit = M.finding_limit(want, dtype)
    assert (np.abs(want).max(-1) > 0.5).all()                    # every row finds something

    def out_of_bounds(**how):
        wrong = M.found(q, k, v, bits, q_lens, kv_lens, scale, **{**dict(window=window, sinks=sinks, held=as_held), **how})
        return (np.abs(wrong - want) > 2 * limit).any()

    def units_reversed(x, b):
        x = x.copy()
        for a in range(0, len(x), 32):
            x[a:a + 32] = x[a:a + 32][::-1].copy()
        return x

    assert out_of_bounds(held=units_reversed) or max(kv_lens) == 1
    assert out_of_bounds(held=lambda x, b: x * 1.02)
    assert out_of_bounds(held=lambda x, b: np.roll(x, 1, 0))
    assert out_of_bounds(seen=MISTAKES["the last token"])
    if window:
        assert out_of_bounds(window=window + 1) or kv_lens[0] <= window
    heads_swapped = M.found(q[:, ::-1], k, v, bits, q_lens, kv_lens, scale, window, sinks, held=as_held)
    assert (np.abs(heads_swapped - want) > 2 * limit).any()


@pytest.mark.parametrize("n,window,sinks", [(700, 0, 0), (128, 0, 0), (610, 100, 0), (600, 400, 5)])
@pytest.mark.parametrize("bits", [4, 8])
def test_the_bound_of_a_row_tells_mistakes_in_ordinary_numbers(n, window, sinks, bits):
    """random keys, values and queries by kv_bounds: a unit left out, its values in reverse, values 2 % too large, a window one too large"""
    rng = np.random.default_rng(n)
    q = O.rounded(rng.standard_normal((1, 8, 128)), "bf16")
    k, v = (O.rounded(rng.standard_normal((n, 2, 128)) * rng.uniform(0.3, 2, (2, 128)), "bf16") for _ in "kv")

    def attended(v, window=window, drop=()):
        keep = [t for t in kv_bounds.seen(n - 1, n, window, sinks) if t not in drop]
        out = np.zeros(q.shape)
        for h in range(8):
            x = O.values(k, bits)[keep, h // 4] @ q[0, h].astype(np.float64) * 128 ** -0.5
            w = np.exp(x - x.max())
            out[0, h] = w @ v[keep, h // 4] / w.sum()
        return out

    held = O.values(v, bits)
    want, limit = kv_bounds.attention(q, [k], [v], bits, [1], [n], 128 ** -0.5, "bf16", window, sinks)
    assert np.abs(attended(held) - want).max() < 1e-12
    unit = np.arange(n // 32 * 32 - 32, n // 32 * 32)
    turned = held.copy()
    turned[unit] = held[unit][::-1]
    for wrong in (attended(held, drop=unit), attended(turned)) + ((attended(held, window=window + 1),) if window and window < 200 else ()):
        assert (np.abs(wrong - want) > limit).any()
