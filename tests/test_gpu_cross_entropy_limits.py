"""Linear cross entropy of few rows on either side of the vocabulary sizes from which
its own kernels leave it to the tiles: W repeats a pattern of rows, so 64-bit values of
the pattern give those of millions of entries.

Bounds: each logit as in test_gpu_cross_entropy_range.py; a sum over the vocabulary is
formed in no longer a chain than a 256th of it (dx: slices of K; lse: 64 threads that
merge the tiles, 64 entries each at least)."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb
from test_gpu_cross_entropy_range import DS, U, logits

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

PERIOD = 1021


def inputs(rows, dim, vocab, dt):
    pattern = R.rounded(synth.normal(vocab % 1000 + dim, (PERIOD, dim)), dt)
    x = R.rounded(synth.normal(rows + dim, (rows, dim)), dt)
    t = (synth.uniform01(rows + 1, rows) * vocab).astype(np.int32)
    t[0] = vocab - 1
    if rows > 2:
        t[1], t[2] = -1, 0
    return x, pattern, t, synth.normal(rows + 4, (rows,))


def expected(x, pattern, t, g, vocab, dt):
    """(lse, bound), (loss, bound), (dx, bound), dw's (pattern rows, bound) and what the
    targets add to dw."""
    x, w, g = (np.asarray(a, np.float64) for a in (x, pattern, g))
    count = np.bincount(np.arange(vocab) % PERIOD, minlength=PERIOD).astype(np.float64)
    depth = vocab // 256 + 700
    on = (t >= 0) & (t < vocab)
    at = np.where(on, t, 0) % PERIOD
    i = np.arange(len(t))
    z, ez = logits(x, w, dt)
    m = z.max(1, keepdims=True)
    s = np.exp(z - m) * count
    lse = (m + np.log(s.sum(1, keepdims=True)))[:, 0]
    el = ((ez + 4 * U * (1 + np.abs(z - m))) * s).sum(1) / s.sum(1) + depth * U + 3 * U * np.abs(lse)
    out = [(lse, el), (np.where(on, lse - z[i, at], 0.0), np.where(on, el + ez[i, at] + 2 * U * (np.abs(lse) + np.abs(z[i, at])), 0.0))]
    gg = np.where(on, g, 0.0)[:, None]
    p = np.exp(z - lse[:, None])
    ep = p * (ez + el[:, None] + 8 * U * (1 + np.abs(z) + np.abs(lse)[:, None])) * (1 + DS[dt]) + (DS[dt] + 2 * U) * p + R.NORMAL
    target = np.abs(gg) * np.abs(w[at]) * np.where(on, 1.0, 0.0)[:, None]
    dx = (p * gg * count) @ w - gg * w[at]
    e = (ep * np.abs(gg) * count) @ np.abs(w) + depth * U * ((p * np.abs(gg) * count) @ np.abs(w) + target) + (DS[dt] + 4 * U) * target
    out.append((dx, e * (1 + R.HALF[dt]) + R.HALF[dt] * np.abs(dx) + R.TINY[dt]))
    dw = (p * gg).T @ x
    e = (ep * np.abs(gg)).T @ np.abs(x) + (len(t) + 8) * U * ((p * np.abs(gg)).T @ np.abs(x))
    out.append((dw, e * (1 + R.HALF[dt]) + R.HALF[dt] * np.abs(dw) + R.TINY[dt]))
    return out, on, gg


def loss_of(x, pattern, t, vocab, dt):
    X, W, T = R.Dev(x, dt), R.Dev(np.resize(pattern, (vocab, x.shape[1])), dt), R.Dev(t, abi.I32)
    L, S = R.Dev(shape=(len(x),)), R.Dev(shape=(len(x),))
    hb.linear_cross_entropy(dt, X.ptr, W.ptr, T.ptr, L.ptr, S.ptr, *x.shape, vocab)
    hb.synchronize()
    return X, W, T, L, S


@pytest.mark.parametrize("dt,rows,dim,vocab", [(abi.F32, 3, 5, 1 << 24), (abi.BF16, 3, 5, 1 << 24), (abi.F16, 16, 3, 1 << 24),
                                               (abi.F32, 20, 6, 1 << 23), (abi.F32, 40, 4, 1 << 22)])
@pytest.mark.parametrize("more", [0, 77])
def test_gradients_on_either_side_of_the_bytes_of_dS(dt, rows, dim, vocab, more):
    vocab += more
    x, pattern, t, g = inputs(rows, dim, vocab, dt)
    X, W, T, L, S = loss_of(x, pattern, t, vocab, dt)
    G, DX, DW = R.Dev(g), R.Dev(dt=dt, shape=x.shape), R.Dev(dt=dt, shape=(vocab, dim))
    hb.linear_cross_entropy_vjp(dt, X.ptr, W.ptr, T.ptr, S.ptr, G.ptr, DX.ptr, DW.ptr, rows, dim, vocab)
    hb.synchronize()
    (lse, loss, dx, dw), on, gg = expected(x, pattern, t, g, vocab, dt)
    R.check(S.get(), *lse, "lse")
    R.check(L.get(), *loss, "loss")
    R.check(DX.get(), *dx, "dx")
    got = DW.get()
    hit = np.unique(t[on])
    full = dw[0][hit % PERIOD].copy()
    np.subtract.at(full, np.searchsorted(hit, t[on]), (gg * np.asarray(x, np.float64))[on])
    size = np.zeros_like(full)
    np.add.at(size, np.searchsorted(hit, t[on]), np.abs(gg * x)[on])
    R.check(got[hit], full, 2 * dw[1][hit % PERIOD] + (DS[dt] + (rows + 8) * U + 2 * R.HALF[dt]) * (size + np.abs(full)), "dw of targets")
    got[hit] = dw[0][hit % PERIOD]
    for k in range(0, vocab, 1 << 20):
        part = got[k:k + (1 << 20)]
        i = np.arange(k, k + len(part)) % PERIOD
        assert (np.abs(part - dw[0][i]) <= dw[1][i]).all(), k


@pytest.mark.parametrize("dt,rows", [(abi.F32, 128), (abi.BF16, 64), (abi.F32, 2)], ids=["f32", "bf16", "f32 by entries"])
@pytest.mark.parametrize("more", [0, 77])
def test_losses_on_either_side_of_the_bytes_of_statistics(dt, rows, more):
    """And, of two rows, of the entries that a launch can count."""
    vocab = min((1 << 33) // rows, 1 << 29) + more
    x, pattern, t, g = inputs(rows, 1, vocab, dt)
    _, _, _, L, S = loss_of(x, pattern, t, vocab, dt)
    (lse, loss, _, _), _, _ = expected(x, pattern, t, g, vocab, dt)
    R.check(S.get(), *lse, "lse")
    R.check(L.get(), *loss, "loss")
