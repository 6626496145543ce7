"""Layer norm with weight and bias where the mean is far above the deviations:
the f32 mean's own error (its rounding and its sum's) must not be in the result.

Bounds (u = 2^-24, D the depth of a row's sum): the mean is off by D u of the mean
magnitude, the mean of the deviations from it, which is taken off again, by D u of
their mean magnitude, that first error among it: D u mean|x - mean| +
2 (D u)^2 mean|x| is left. The variance is off by as much of itself and of the square
of the mean's error. The rest as in operators_ref.py."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from test_gpu_norm_affine import EPS, inputs, run

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

U = R.U


def expected(x, dy, w, b, dt):
    """[(y, bound), (dx, bound), (dw, bound), (db, bound)]."""
    x, dy, w, b = (np.asarray(a, np.float64) for a in (x, dy, w, b))
    rows, cols = x.shape
    d = R._row_depth(cols) + 2
    xc = x - x.mean(1, keepdims=True)
    var = (xc ** 2).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(var + EPS)
    xh = xc * rstd
    moved = d * U * np.abs(x).mean(1, keepdims=True)          # the mean's error
    rel = d * U * (var + 2 * moved ** 2) / (var + EPS) + 8 * U  # rstd's, twice over
    e = rstd * d * U * (np.abs(xc).mean(1, keepdims=True) + 2 * moved) + rel * np.abs(xh)
    y = xh * w + b
    out = [(y, np.abs(w) * e + 2 * U * (np.abs(xh * w) + np.abs(y)))]
    g = dy * w
    c1, c2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    dx = rstd * (g - c1 - xh * c2)
    m = np.abs(g).mean(1, keepdims=True)
    # mean(g xh) is of g d, less the mean of d times that of g: both products' errors.
    e2 = (d + 6) * U * ((np.abs(g * xh)).mean(1, keepdims=True) + 2 * rstd * moved * m) + (np.abs(g) * e).mean(1, keepdims=True)
    terms = np.abs(g) + np.abs(c1) + np.abs(xh * c2)
    out.append((dx, rstd * (4 * U * terms + (d + 2) * U * m + np.abs(xh) * e2 + e * np.abs(c2) + e * e2) + rel * rstd * terms))
    groups = 256 if cols <= 16384 else 64
    n = rows // groups + 1 + 4 + groups // 8 + 8
    out.append(((dy * xh).sum(0), (n + 2) * U * np.abs(dy * xh).sum(0) + (np.abs(dy) * e).sum(0)))
    out.append((dy.sum(0), n * U * np.abs(dy).sum(0)))
    return [(v, b * (1 + R.HALF[dt]) + R.HALF[dt] * np.abs(v) + R.TINY[dt]) for v, b in out]


COLS = [3, 64, 100, 777, 1500, 4096, 9001, 17000]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("cols", COLS)
def test_constant_rows(cols, dt):
    """No deviations: y = b, whatever the row's value."""
    x, dy, w, b = inputs(6, cols, dt)
    x[:] = R.rounded(np.array([3000.7, -0.1, 1234.567, 1e-3, -777.77, 1 / 3], np.float32), dt)[:, None]
    for name, a, (v, bound) in zip(("y", "dx", "dw", "db"), run(x, dy, w, b, dt), expected(x, dy, w, b, dt)):
        R.check(a, v, bound, f"{name} of constant rows of {cols}")


@pytest.mark.parametrize("mean", [3000.0, -50000.0])
@pytest.mark.parametrize("cols", COLS)
def test_a_mean_far_above_the_deviations(cols, mean):
    x, dy, w, b = inputs(5, cols, abi.F32, mean=mean)
    for name, a, (v, bound) in zip(("y", "dx", "dw", "db"), run(x, dy, w, b, abi.F32), expected(x, dy, w, b, abi.F32)):
        R.check(a, v, bound, f"{name} around {mean}, {cols} columns")


@pytest.mark.parametrize("cols", [64, 1500, 17000])
def test_squares_past_the_range(cols):
    """Deviations whose squares are infinite have no f32 variance: rstd is 0 and y
    is b, dx 0."""
    x, dy, w, b = inputs(3, cols, abi.F32)
    x *= np.float32(1e30)
    y, dx, dw, _ = run(x, dy, w, b, abi.F32)
    np.testing.assert_array_equal(y, np.broadcast_to(b.astype(np.float64), y.shape))
    assert not dw.any() and not dx.any()
