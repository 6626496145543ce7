"""Linear cross entropy on operands whose sizes differ widely, and with
infinities: each result against 64 bits within a bound made from its own row's and
column's terms, whatever the rest of the operands hold.

Bounds (u = 2^-24). A logit is a sum of dim terms in f32, of operands that are
exact (16 bits) or have 22 bits and, below 2^-18 of their own row's largest
value, what is left of 2^-39 of that (f32). dS is held to 24 bits (f32), 16 (bf16: two
planes, half of 2^-7 of half of 2^-7) or 22 with a floor of 2^-40 of dloss (f16: two planes
of dS / dloss times 2^15, half of f16's smallest step); its sums are f32; f16's
dloss x is held alike, with a floor of 2^-39 of the largest, and products of the
second planes, 2^-22 of a term, are left out; a result is rounded once."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from test_gpu_cross_entropy import inputs, run

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

U = R.U
DS = {abi.F32: 2.0 ** -24, abi.BF16: 2.0 ** -16, abi.F16: 2.0 ** -22}


def logits(x, w, dt):
    z = x @ w.T
    e = (x.shape[1] + 8) * U * (np.abs(x) @ np.abs(w).T)
    if dt == abi.F32:
        a, b = np.abs(x), np.abs(w)
        e = e + 2.0 ** -39 * (a.max(1)[:, None] * b.sum(1) + a.sum(1)[:, None] * b.max(1))
    return z, e


def forward(x, w, t, dt):
    """[(loss, bound), (lse, bound)]."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    z, ez = logits(x, w, dt)
    lse, el = R._lse(z, ez)
    on = (t >= 0) & (t < len(w))
    i, at = np.arange(len(t)), np.where(on, t, 0)
    loss = np.where(on, lse - z[i, at], 0.0)
    return [(loss, np.where(on, el + ez[i, at] + 2 * U * (np.abs(lse) + np.abs(z[i, at])), 0.0)), (lse, el)]


def backward(x, w, t, dloss, dt):
    """[(dx, bound), (dw, bound)] with the kernel's own lse."""
    x, w, g = (np.asarray(a, np.float64) for a in (x, w, dloss))
    on = (t >= 0) & (t < len(w))
    x = np.where(on[:, None], x, 0.0)
    z, ez = logits(x, w, dt)
    lse, el = R._lse(z, ez)
    p = np.exp(z - lse[:, None])
    ep = p * (ez + el[:, None] + 8 * U * (1 + np.abs(z) + np.abs(lse)[:, None]))
    p[np.arange(len(t))[on], t[on]] -= 1
    ep += 2 * U * np.abs(p) + R.NORMAL
    gg = np.where(on, g, 0.0)[:, None]
    ds = p * gg
    eds = (ep + 2 * U * np.abs(p)) * np.abs(gg) * (1 + DS[dt]) + DS[dt] * np.abs(ds) + R.NORMAL * (gg != 0)
    if dt == abi.F16:
        eds = eds + 2.0 ** -40 * np.abs(gg)
    out = []
    for a, ea, m in ((ds, eds, w), (ds.T, eds.T, x)):
        v = a @ m
        e = ((a.shape[1] + 8) * U) * ((np.abs(a) + ea) @ np.abs(m)) + ea @ np.abs(m)
        if dt == abi.F16 and m is x:
            e = e + 2.0 ** -21 * (np.abs(a) @ np.abs(m)) + 2.0 ** -39 * np.abs(gg * x).max() * np.abs(p).sum(0)[:, None]
        out.append((v, e * (1 + R.HALF[dt]) + R.HALF[dt] * np.abs(v) + R.TINY[dt]))
    return out


def check_all(got, x, w, t, g, dt):
    for name, a, (v, b) in zip(("loss", "lse", "dx", "dw"), got, forward(x, w, t, dt) + backward(x, w, t, g, dt)):
        R.check(a, v, b, name)


ROWS = [5, 17, 50, 65, 129, 300]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,dim,vocab", [(17, 72, 700), (65, 77, 515), (130, 70, 1025), (300, 264, 777), (700, 64, 333)])
def test_gradients_lose_nothing_to_dS(rows, dim, vocab, dt):
    """16-bit gradients are off by their own rounding and no more: dS holds
    more bits than they do."""
    a = inputs(rows, dim, vocab, dt)
    check_all(run(*a, dt), *a, dt)


@pytest.mark.parametrize("rows", ROWS)
def test_a_vocabulary_entry_far_above_the_others(rows):
    """One row of w is 2^30 times the others (its logit is -2^30, its
    probability 0): the others keep their digits."""
    x, w, t, g = inputs(rows, 72, 700, abi.F32)
    x[:, 3] = 1.0
    w[:, 3] *= 0.125
    t[t == 11] = 12
    w[11] = 0.0
    w[11, 3] = -2.0 ** 30
    got = run(x, w, t, g, abi.F32)
    want = forward(x, w, t, abi.F32) + backward(x, w, t, g, abi.F32)
    for name, a, (v, b) in zip(("loss", "lse"), got, want):
        R.check(a, v, b, name)
    keep = np.arange(72) != 3   # column 3 of dx is bounded by 0 times 2^30
    R.check(got[2][:, keep], want[2][0][:, keep], want[2][1][:, keep], "dx")
    R.check(got[3], *want[3], "dw")


@pytest.mark.parametrize("dt", [abi.F32, abi.BF16], ids=R.NAMES.get)
@pytest.mark.parametrize("rows", ROWS)
def test_a_row_far_above_the_others(rows, dt):
    """One row of x holds 2^30 where w has zeros: its own gradients aside, the
    others' are what they were."""
    x, w, t, g = inputs(rows, 72, 700, dt, ignored=0.0)
    w[:, 5] = 0.0
    x[2, 5] = 2.0 ** 30
    check_all(run(x, w, t, g, dt), x, w, t, g, dt)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows", ROWS)
def test_a_dloss_far_above_the_others(rows, dt):
    x, w, t, g = inputs(rows, 72, 700, dt, ignored=0.0)
    g[1] = 2.0 ** 12 if dt == abi.F16 else 2.0 ** 30
    if dt == abi.F16:
        g[2:] *= 2.0 ** -6
    check_all(run(x, w, t, g, dt), x, w, t, g, dt)


@pytest.mark.parametrize("dt", [abi.F32, abi.BF16], ids=R.NAMES.get)
@pytest.mark.parametrize("rows", ROWS)
def test_improbable_words_keep_their_digits(rows, dt):
    """A third of the vocabulary at logits 40 below the others, probabilities
    of 2^-58: those rows of dw are as exact as the others for their size."""
    x, w, t, g = inputs(rows, 72, 700, dt)
    x[:, 7] = 8.0
    w[:, 7] = 0.0
    w[::3, 7] = -5.0
    t = np.where((t >= 0) & (t < 700) & (t % 3 == 0), t + 1, t).astype(np.int32)
    check_all(run(x, w, t, g, dt), x, w, t, g, dt)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dim", [72, 77])
def test_an_entry_ruled_out_by_an_infinity(rows, dim, dt):
    """-inf in one row of w where x is positive: that logit is -inf, its
    probability 0, and losses and gradients are those without the entry; dx is NaN
    in the infinity's column (0 times infinity), rows without a target have no
    gradient all the same."""
    vocab = 515
    x, w, t, g = inputs(rows, dim, vocab, dt)
    x[:, 4] = 0.5 + np.abs(x[:, 4])
    x = R.rounded(x, dt)
    t[t == vocab - 1] = 3
    w[vocab - 1, 4] = -np.inf
    t[t == vocab] = -1
    t[0] = 3
    t[1] = -100
    got = run(x, w, t, g, dt)
    want = forward(x, w[:-1], t, dt) + backward(x, w[:-1], t, g, dt)
    R.check(got[0], *want[0], "loss")
    R.check(got[1], *want[1], "lse")
    on = (t >= 0) & (t < vocab)
    keep = np.arange(dim) != 4
    R.check(got[2][:, keep], want[2][0][:, keep], want[2][1][:, keep], "dx")
    assert np.isnan(got[2][on, 4]).all() and not got[2][~on].any()
    R.check(got[3][:-1], *want[3], "dw")
    assert not got[3][-1].any()


@pytest.mark.parametrize("rows", ROWS)
def test_values_next_to_the_largest_one(rows):
    """f32 values that fewer bits would round to infinity, where x has zeros:
    nothing but the sums over them (column 6 of dx) may leave the range."""
    x, w, t, g = inputs(rows, 72, 300, abi.F32)
    x[:, 6] = 0.0
    w[5, 6] = np.finfo(np.float32).max
    w[6, 6] = -np.finfo(np.float32).max
    got = run(x, w, t, g, abi.F32)
    got[2] = got[2][:, np.arange(72) != 6]
    for name, a in zip(("loss", "lse", "dx", "dw"), got):
        assert np.isfinite(a).all(), name
