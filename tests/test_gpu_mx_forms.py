"""Products of microscaled numbers in every form of their kernels: results of each type, biases and residuals, rows of longer ones.  Operands are whole
codes, sums multiples of 1/4 that 32 bits hold in any order, so that a result is the definition's, rounded once to its type: bit for bit."""
import numpy as np
import pytest

import mx_forms
import mx_oracle as O
from test_gpu_mx import Part, matrix, part_of
from tpu_compiler_amd import capi, mx
from tpu_compiler_amd.kv_cache import DeviceArray

pytestmark = pytest.mark.gpu
TABLE = O.VALUES.astype(np.float32)


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context()
    yield c
    c.close()


def codes_of(rng, rows, cols):
    """codes of any kind, zeros behind the last column; scales of 1; their values in 32 bits"""
    blocks = -(-cols // 32)
    c = rng.integers(0, 16, (rows, blocks * 32), np.uint8)
    c[:, cols:] = 0
    return c[:, 0::2] | c[:, 1::2] << 4, np.full((rows, blocks), 127, np.uint8), TABLE[c[:, :cols]]


def part_matrix(ctx, codes, scales, cols):
    """a matrix whose rows are parts of longer ones, between which are scales that make NaN of whatever they belong to"""
    c, s = (DeviceArray.of(ctx, np.pad(v, ((0, 0), (p, q)), constant_values=255), "u8") for v, p, q in ((codes, 16, 32), (scales, 1, 2)))
    return mx.MXMatrix(ctx, len(codes), cols, Part(c, codes.shape, (codes.shape[1] + 48, 1), 16), Part(s, scales.shape, (scales.shape[1] + 3, 1), 1))


def results(ctx, rows, cols, n):
    """each type's, of x in 4 bits and as elements, w and x by themselves and as parts of longer rows, with and without a bias and a residual"""
    rng = np.random.default_rng(rows + cols + n)
    x, w = codes_of(rng, rows, cols), codes_of(rng, n, cols)
    # no sum of some of the terms is larger than all their sizes; with the bias and the residual, in units of 1/4
    assert (np.abs(x[2]) @ np.abs(w[2]).T).max() + 10 + 128 < 2 ** 24 / 4
    want = x[2] @ w[2].T
    bias = rng.integers(-40, 41, n).astype(np.float32) / 4
    more = rng.integers(-128, 129, (rows, n)).astype(np.float32)      # that every type holds
    bias_d = DeviceArray.of(ctx, bias, "f32")
    arrays = [matrix(ctx, *w[:2], cols), part_matrix(ctx, *w[:2], cols), matrix(ctx, *x[:2], cols), part_matrix(ctx, *x[:2], cols)]
    for dtype in ("bf16", "f16", "f32"):
        elements = None
        if rows * cols < 4e6:
            elements, base = part_of(ctx, x[2], dtype, 9, 1, fill=np.nan)
            arrays.append(base)
        # (x, w, bias, residual: in the result's place, by itself, or none)
        calls = [(arrays[2], arrays[0], None, None), (arrays[3], arrays[1], bias_d, "here"), (elements, arrays[1], bias_d, "here"), (elements, arrays[0], None, "there"),
                 (arrays[2], arrays[1], None, "there"), (arrays[3], arrays[0], bias_d, None)]
        for a, b, bias_a, residual in calls:
            if a is None:
                continue
            out, whole = part_of(ctx, more if residual == "here" else np.full((rows, n), 3.0), dtype, 5, 3)
            there = DeviceArray.of(ctx, more, dtype) if residual == "there" else None
            mx.product(ctx, a, b, out, bias_a, out if residual == "here" else there)
            expected = want if bias_a is None else want + bias
            expected = O.rounded(expected if residual is None else expected + more, dtype)
            got = whole.numpy()[3:].reshape(rows, n + 5).astype(np.float32)
            assert np.array_equal(got[:, :n], expected), (dtype, a is elements, bias_a is not None, residual)
            assert (got[:, n:] == 7).all() and (whole.numpy()[:3] == 7).all()
            whole.free()
            if there is not None:
                there.free()
    for m in arrays + [bias_d]:
        if isinstance(m, mx.MXMatrix):
            for part in (m.codes, m.scales):
                getattr(part, "base", part).free()
        else:
            m.free()


@pytest.mark.parametrize("form,parts,rows,cols,n", mx_forms.CASES)
def test_results_of_tiles(ctx, form, parts, rows, cols, n):
    results(ctx, rows, cols, n)


@pytest.mark.parametrize("waves,groups,rows,cols,n", mx_forms.FEW_CASES)
def test_results_of_few_rows(ctx, waves, groups, rows, cols, n):
    results(ctx, rows, cols, n)
