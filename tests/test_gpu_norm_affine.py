"""Layer norm with weight and bias, and its gradients, against 64 bits, within
the bounds of operators_ref.py."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

EPS = 1e-5


def inputs(rows, cols, dt, mean=0.5, seed=0):
    x = synth.normal(7 * rows + cols + seed, (rows, cols), mean, 2.0)
    dy = synth.normal(11 * rows + cols + seed, (rows, cols))
    w, b = synth.normal(cols + 1, (cols,), 1.0, 0.2), synth.normal(cols + 2, (cols,), 0.0, 0.2)
    return [R.rounded(a, dt) for a in (x, dy, w, b)]


def run(x, dy, w, b, dt, offset=0, stream=None):
    rows, cols = x.shape
    X, DY, W, B = (R.Dev(a, dt, offset) for a in (x, dy, w, b))
    Y, DX = (R.Dev(dt=dt, offset=offset, shape=x.shape) for _ in range(2))
    DW, DB = (R.Dev(dt=dt, offset=offset, shape=(cols,)) for _ in range(2))
    hb.layernorm_affine_rows(dt, X.ptr, W.ptr, B.ptr, Y.ptr, rows, cols, EPS, stream)
    hb.layernorm_affine_vjp_rows(dt, DY.ptr, X.ptr, W.ptr, DX.ptr, DW.ptr, DB.ptr, rows, cols, EPS, stream)
    hb.synchronize(stream)
    return [t.get() for t in (Y, DX, DW, DB)]


def check_all(got, x, dy, w, b, dt, what):
    y, bound = R.layer_norm(x, w, b, EPS, dt)
    R.check(got[0], y, bound, f"y {what}")
    for name, g, (v, bd) in zip(("dx", "dw", "db"), got[1:], R.layer_norm_vjp(dy, x, w, EPS, dt)):
        R.check(g, v, bd, f"{name} {what}")


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 64), (9, 255), (4, 256), (6, 257), (1000, 41), (7, 511), (5, 512), (4, 513),
          (3, 768), (33, 777), (3, 1000), (2, 1024), (3, 1025), (5, 2047), (2, 2049), (3, 3001), (2, 4096), (2, 4097),
          (3, 8191), (1, 8200), (2, 12289), (1, 16384), (3, 16385), (2, 20001), (70, 17000), (300, 1024), (600, 4096)]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_matches_64_bits(rows, cols, dt):
    print(f"layer norm {rows}x{cols} {R.NAMES[dt]}", flush=True)
    a = inputs(rows, cols, dt)
    check_all(run(*a, dt), *a, dt, f"{rows}x{cols}")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,cols,offset", [(3, 777, 1), (5, 1024, 3), (2, 4098, 7), (3, 16386, 1), (4, 8, 5)])
def test_any_element_alignment(rows, cols, offset, dt):
    a = inputs(rows, cols, dt)
    check_all(run(*a, dt, offset), *a, dt, f"{rows}x{cols}+{offset}")


@pytest.mark.parametrize("cols", [100, 4096, 17000])
def test_a_large_mean_costs_no_digits_of_the_deviations(cols):
    """Rows of 3000 +- 2: the sums are of deviations from the mean, so the
    bound's only large term is the mean's own rounding."""
    a = inputs(4, cols, abi.F32, mean=3000.0)
    check_all(run(*a, abi.F32), *a, abi.F32, f"mean 3000, {cols}")


@pytest.mark.parametrize("cols", [64, 1500, 17000])
def test_constant_rows_and_non_finite_ones(cols):
    x, dy, w, b = inputs(6, cols, abi.F32)
    x[1] = 4.0               # no variance: xh = 0, y = b
    x[3, cols // 2] = np.nan  # NaN and infinity stay in their rows
    x[4, 0] = np.inf
    got = run(x, dy, w, b, abi.F32)
    np.testing.assert_array_equal(got[0][1], b.astype(np.float64))
    assert np.isnan(got[0][3:5]).all() and np.isnan(got[1][3:5]).all()
    fine = [0, 1, 2, 5]
    y, bound = R.layer_norm(x[fine], w, b, EPS, abi.F32)
    R.check(got[0][fine], y, bound, "y of the finite rows")
    dx, bd = R.layer_norm_vjp(dy[fine], x[fine], w, EPS, abi.F32)[0]
    R.check(got[1][fine], dx, bd, "dx of the finite rows")
    db, bd = R.layer_norm_vjp(dy, np.where(np.isfinite(x), x, 0), w, EPS, abi.F32)[2]
    R.check(got[3], db, bd, "db")


def test_no_rows():
    DW, DB = R.Dev(dt=abi.BF16, shape=(40,)), R.Dev(dt=abi.BF16, shape=(40,))
    hb.layernorm_affine_rows(abi.BF16, 0, 0, 0, 0, 0, 40, EPS)
    hb.layernorm_affine_vjp_rows(abi.BF16, 0, 0, 0, 0, DW.ptr, DB.ptr, 0, 40, EPS)
    hb.synchronize()
    assert not DW.get().any() and not DB.get().any()


@pytest.mark.parametrize("cols", [96, 5000])
def test_gradient_against_differences(cols):
    """(f(x + h d) - f(x - h d)) / 2h of the 64-bit forward for f = sum(dy y):
    the gradient's inner product with d, for a direction in x, w and b. The
    differences' own error is of the order of h^2 times third derivatives:
    under 1e-6 of the terms at h = 1e-4."""
    x, dy, w, b = inputs(5, cols, abi.F32)
    got = run(x, dy, w, b, abi.F32)
    h = 1e-4
    want = R.layer_norm_vjp(dy, x, w, EPS, abi.F32)
    for i, (at, g, (v, bound)) in enumerate(zip((0, 2, 3), got[1:], want)):
        d = synth.normal(50 + i, g.shape)
        plus, minus = [x, dy, w, b], [x, dy, w, b]
        plus[at] = plus[at].astype(np.float64) + h * d
        minus[at] = minus[at].astype(np.float64) - h * d
        f = [(R.layer_norm(a[0], a[2], a[3], EPS, abi.F32)[0] * dy).sum() for a in (plus, minus)]
        slope, inner = (f[0] - f[1]) / (2 * h), (g * d).sum()
        assert abs(slope - inner) <= 1e-6 * np.abs(v * d).sum() + (np.abs(d) * bound).sum(), (i, slope, inner)


def test_same_bits_every_time_and_on_another_stream():
    a = inputs(700, 1024, abi.BF16)
    one = run(*a, abi.BF16)
    s = hb.create_stream()
    try:
        for stream in (None, s):
            for x, y in zip(one, run(*a, abi.BF16, stream=stream)):
                np.testing.assert_array_equal(x, y)
    finally:
        hb.destroy_stream(s)
