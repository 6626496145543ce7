"""Linear cross entropy and its gradients against 64 bits, within the bounds of
operators_ref.py."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


def inputs(rows, dim, vocab, dt, ignored=0.25, spread=1.0):
    """Logits of spread about 1, the target's raised; a share of the rows ignored."""
    w = R.rounded(synth.normal(vocab + dim, (vocab, dim), 0.0, spread / dim ** 0.5), dt)
    t = (synth.uniform01(rows + 1, rows) * vocab).astype(np.int32)
    x = synth.normal(rows + dim, (rows, dim)) + 12 * synth.uniform01(rows + 2, rows)[:, None].astype(np.float32) * w[t]
    skip = synth.uniform01(rows + 3, rows) < ignored
    t[skip] = np.where(np.arange(skip.sum()) % 2, -100, vocab)
    dloss = np.where(np.arange(rows) % 3 == 2, 0.125, synth.normal(rows + 4, (rows,))).astype(np.float32)
    return R.rounded(x, dt), w, t, dloss


def run(x, w, t, dloss, dt, offset=0, stream=None, want="xw"):
    (rows, dim), vocab = x.shape, len(w)
    X, W, T, G = R.Dev(x, dt, offset), R.Dev(w, dt, offset), R.Dev(t, abi.I32), R.Dev(dloss)
    L, S = R.Dev(shape=(rows,)), R.Dev(shape=(rows,))
    DX, DW = R.Dev(dt=dt, offset=offset, shape=x.shape), R.Dev(dt=dt, offset=offset, shape=w.shape)
    hb.linear_cross_entropy(dt, X.ptr, W.ptr, T.ptr, L.ptr, S.ptr, rows, dim, vocab, stream)
    hb.linear_cross_entropy_vjp(dt, X.ptr, W.ptr, T.ptr, S.ptr, G.ptr, DX.ptr if "x" in want else None,
                                DW.ptr if "w" in want else None, rows, dim, vocab, stream)
    hb.synchronize(stream)
    return [a.get() for a in (L, S)] + [a.get() if k in want else None for k, a in (("x", DX), ("w", DW))]


def check_all(got, x, w, t, dloss, dt, what):
    for name, g, (v, b) in zip(("loss", "lse", "dx", "dw"), got,
                               R.cross_entropy(x, w, t, dt) + R.cross_entropy_vjp(x, w, t, dloss, dt)):
        if g is not None:
            R.check(g, v, b, f"{name} {what}")


SIZES = [(1, 1, 1), (1, 8, 2), (2, 3, 5), (5, 64, 1), (1, 64, 1000), (7, 33, 37), (8, 768, 1003), (16, 128, 256),
         (16, 2011, 130), (17, 100, 257), (32, 200, 321), (33, 32, 4099), (40, 2, 70), (64, 96, 512), (65, 333, 190), (100, 256, 300), (128, 64, 128), (128, 261, 777), (129, 70, 1025),
         (256, 256, 512), (257, 40, 2001), (300, 520, 777), (513, 288, 1536), (1000, 77, 3203)]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,dim,vocab", SIZES)
def test_matches_64_bits(rows, dim, vocab, dt):
    print(f"cross entropy {rows}x{dim} over {vocab} {R.NAMES[dt]}", flush=True)
    a = inputs(rows, dim, vocab, dt)
    check_all(run(*a, dt), *a, dt, f"{rows}x{dim}x{vocab}")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,dim,vocab,offset", [(9, 64, 300, 1), (130, 77, 515, 3), (300, 128, 1000, 5)])
def test_any_element_alignment(rows, dim, vocab, offset, dt):
    a = inputs(rows, dim, vocab, dt)
    check_all(run(*a, dt, offset), *a, dt, f"+{offset}")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows", [5, 40, 300])
def test_rows_without_a_target(rows, dt):
    """Whatever x and dloss hold there: loss 0, dx 0, nothing in dw; with no
    row left all gradients are 0."""
    x, w, t, g = inputs(rows, 72, 700, dt, ignored=0.0)
    clean = x.copy()
    t[1::3] = (-1, 700, np.iinfo(np.int32).min, np.iinfo(np.int32).max)[rows % 4]
    off = (t < 0) | (t >= 700)
    x[off] = np.nan
    x[off, 0] = np.inf
    g[off] = np.nan
    got = run(x, w, t, g, dt)
    want = R.cross_entropy(clean, w, t, dt) + R.cross_entropy_vjp(clean, w, t, np.where(off, 0, g), dt)
    assert not got[0][off].any() and not got[2][off].any()
    R.check(got[0], *want[0], "loss")
    R.check(got[1][~off], want[1][0][~off], want[1][1][~off], "lse")
    R.check(got[2], *want[2], "dx")
    R.check(got[3], *want[3], "dw")
    t[:] = -100
    got = run(x, w, t, g, dt)
    assert not got[0].any() and not got[2].any() and not got[3].any()


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows", [3, 50, 260])
def test_far_apart_logits(rows, dt):
    """Logits of some thousands: one probability of 1 and the rest 0, or far
    beyond the range of exp without the maximum taken off."""
    x, w, t, g = inputs(rows, 64, 333, dt, spread=100.0)
    check_all(run(x, w, t, g, dt), x, w, t, g, dt, "spread 100")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows", [3, 260])
def test_far_apart_logits_with_other_targets(rows, dt):
    """As above with targets that are not the largest logit: losses of
    thousands, gradients of -1 and 1."""
    x, w, t, g = inputs(rows, 64, 333, dt, spread=100.0)
    t = np.where(t >= 0, (t + 5) % 333, t).astype(np.int32)
    check_all(run(x, w, t, g, dt), x, w, t, g, dt, "spread 100, other targets")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,dim", [(5, 64), (50, 77), (270, 264)])
def test_values_of_very_different_size(rows, dim, dt):
    """Elements, rows and dloss over some twenty binary orders of magnitude
    (f32 and f16 hold their small parts scaled), a vocabulary entry that is all
    zeros, and rows without a target that hold huge values."""
    vocab = 515
    x, w, t, g = inputs(rows, dim, vocab, dt)
    spread = lambda seed, shape, n: np.exp2(-np.floor(n * synth.uniform01(seed, int(np.prod(shape))))).reshape(shape)
    x = R.rounded((x * spread(1, (rows, 1), 6) * spread(2, (rows, dim), 8)).astype(np.float32), dt)
    w = R.rounded((w * spread(3, (vocab, 1), 6) * spread(4, (vocab, dim), 8)).astype(np.float32), dt)
    w[3] = 0.0
    x[0] = 0.0
    t[0] = 3
    g = (g * spread(5, (rows,), 12)).astype(np.float32)
    off = (t < 0) | (t >= vocab)
    if dt != abi.F16:
        x[off] *= 2.0 ** 60
    got = run(x, w, t, g, dt)
    fine = ~off
    want = R.cross_entropy(x[fine], w, t[fine], dt)
    R.check(got[0][fine], *want[0], "loss")
    R.check(got[1][fine], *want[1], "lse")
    for name, a, b in zip(("dx", "dw"), got[2:], R.cross_entropy_vjp(x, w, t, g, dt)):
        R.check(a, *b, name)


@pytest.mark.parametrize("rows", [4, 300])
def test_non_finite_rows_stay_in_their_rows(rows):
    """NaN and infinity in x of counted rows: NaN loss, lse and dx there and
    nowhere else (dw sums over rows and is NaN)."""
    x, w, t, g = inputs(rows, 64, 300, abi.BF16, ignored=0.0)
    x[1] = np.nan
    got = run(x, w, t, g, abi.BF16)
    fine = np.arange(rows) != 1
    want = R.cross_entropy(x[fine], w, t[fine], abi.BF16) + R.cross_entropy_vjp(x[fine], w, t[fine], g[fine], abi.BF16)
    assert np.isnan(got[0][1]) and np.isnan(got[1][1]) and np.isnan(got[2][1]).all()
    for a, b in zip(got[:3], want[:3]):
        R.check(a[fine], *b, "finite rows")


@pytest.mark.parametrize("dt", [abi.F32, abi.BF16], ids=R.NAMES.get)
@pytest.mark.parametrize("rows,dim,vocab", [(9000, 8, 5000), (40000, 16, 3000)])
def test_several_pieces_of_the_vocabulary(rows, dim, vocab, dt):
    a = inputs(rows, dim, vocab, dt)
    check_all(run(*a, dt), *a, dt, f"{rows}x{dim}x{vocab}")


@pytest.mark.parametrize("dt", [abi.F32, abi.BF16], ids=R.NAMES.get)
@pytest.mark.parametrize("vocab", [1 << 22, (1 << 22) + 77])
def test_few_rows_of_millions_of_entries(vocab, dt):
    """Either side of the vocabulary that the few rows' own kernels take."""
    a = inputs(3, 8, vocab, dt)
    check_all(run(*a, dt), *a, dt, f"3x8x{vocab}")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows", [6, 40, 300])
def test_one_gradient_alone(rows, dt):
    a = inputs(rows, 72, 700, dt)
    both = run(*a, dt)
    np.testing.assert_array_equal(run(*a, dt, want="x")[2], both[2])
    np.testing.assert_array_equal(run(*a, dt, want="w")[3], both[3])


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows", [6, 40, 300])
def test_a_cotangent_of_zeros(rows, dt):
    x, w, t, g = inputs(rows, 72, 700, dt)
    got = run(x, w, t, np.zeros_like(g), dt)
    assert not got[2].any() and not got[3].any()


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_no_rows(dt):
    DW = R.Dev(dt=dt, shape=(37, 5), offset=1)
    hb.linear_cross_entropy(dt, 0, 0, 0, 0, 0, 0, 5, 37)
    hb.linear_cross_entropy_vjp(dt, 0, 0, 0, 0, 0, None, DW.ptr, 0, 5, 37)
    hb.synchronize()
    assert not DW.get().any()


def test_gradient_against_differences():
    """(f(x + h d) - f(x - h d)) / 2h of the 64-bit losses, f = sum(dloss loss),
    against the gradients' inner product with d; the differences' error is of
    the order of h^2 times third derivatives, under 1e-6 of the terms."""
    x, w, t, g = inputs(60, 64, 500, abi.F32)
    got, want, h = run(x, w, t, g, abi.F32), R.cross_entropy_vjp(x, w, t, g, abi.F32), 1e-4
    for i in range(2):
        d = synth.normal(70 + i, got[2 + i].shape)
        moved = [(x + s * h * d, w) if i == 0 else (x, w + s * h * d) for s in (1, -1)]
        f = [(R.cross_entropy(*m, t, abi.F32)[0][0] * g).sum() for m in moved]
        slope, inner = (f[0] - f[1]) / (2 * h), (got[2 + i] * d).sum()
        v, b = want[i]
        assert abs(slope - inner) <= 1e-6 * np.abs(v * d).sum() + (np.abs(d) * b).sum(), (i, slope, inner)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_same_bits_every_time_and_on_another_stream(dt):
    a = inputs(300, 264, 1500, dt)
    one = run(*a, dt)
    s = hb.create_stream()
    try:
        for stream in (None, s):
            for x, y in zip(one, run(*a, dt, stream=stream)):
                np.testing.assert_array_equal(x, y)
    finally:
        hb.destroy_stream(s)
