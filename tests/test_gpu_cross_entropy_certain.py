"""Gradients of rows whose target is all but certain: dS of the target is what p misses
to 1, so z has to be the same in the loss and in the gradient, and what is left is the
rounding of lse (of the loss, through lazy streams).

Bound of p - 1 at a target of probability 1 - 2^-33 and less: half a step of lse (32 u
from 32 on, u = 2^-24), and 8 u for the sum of exponentials next to 1, its logarithm
and exp. The sum takes no rounding from the others, which are below u / 2 together."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb
from oxidizedmlx_amd.tensor import Tensor, eval_all, value_and_grad
import test_gpu_cross_entropy as T
from test_gpu_cross_entropy import run

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

U = R.U


def inputs(rows, dim, vocab, dt):
    """Targets' logits of 40 to 60, the others' of spread 2.5 to 4 around 0."""
    w = R.rounded(synth.normal(vocab + dim, (vocab, dim), 0.0, dim ** -0.5), dt)
    t = (synth.uniform01(rows + 1, rows) * vocab).astype(np.int32)
    lift = 40 + 20 * synth.uniform01(rows + 2, rows)
    wt = w[t].astype(np.float64)
    x = R.rounded((lift[:, None] * wt / (wt ** 2).sum(1, keepdims=True)).astype(np.float32), dt)
    return x, w, t, synth.normal(rows + 4, (rows,))


def bounds(x, w, t, g, dt):
    """(dx, bound), (dw, bound)."""
    x, w, g = (np.asarray(a, np.float64) for a in (x, w, g))
    z = x @ w.T
    lse = lse_of(z)
    i = np.arange(len(t))
    rest = np.exp(z - lse[:, None])
    rest[i, t] = 0.0
    assert rest.sum(1).max() < 2.0 ** -33, "not certain"
    p = rest.copy()
    p[i, t] = -rest.sum(1)
    ds = p * g[:, None]
    off = rest * 1e-3   # of probabilities that small more than enough
    off[i, t] = np.spacing(lse.astype(np.float32)).astype(np.float64) / 2 + 8 * U
    off *= np.abs(g)[:, None]
    floor = 2.0 ** -40 if dt == abi.F16 else 0.0
    out = []
    for a, e, m in ((ds, off + floor * np.abs(g)[:, None], w), (ds.T, off.T + floor * np.abs(g), x)):
        v = a @ m
        b = (e @ np.abs(m)) * 1.01 + (a.shape[1] + 8) * U * (np.abs(a) @ np.abs(m))
        out.append((v, b * (1 + R.HALF[dt]) + R.HALF[dt] * np.abs(v) + R.TINY[dt]))
    return out


SIZES = [(5, 256, 1000), (16, 257, 1000), (17, 256, 1000), (40, 256, 1500), (40, 257, 1500), (64, 256, 1000), (65, 260, 1000),
         (100, 256, 2000), (128, 256, 1003), (129, 256, 1000), (300, 256, 2000), (2000, 256, 1500)]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rows,dim,vocab", SIZES)
def test_certain_rows(rows, dim, vocab, dt):
    a = inputs(rows, dim, vocab, dt)
    got = run(*a, dt)
    for name, g, (v, b) in zip(("dx", "dw"), got[2:], bounds(*a, dt)):
        R.check(g, v, b, f"{name} {rows}x{dim}x{vocab}")


@pytest.mark.parametrize("rows,dim,vocab", SIZES)
def test_certain_rows_through_lazy_streams(rows, dim, vocab):
    x, w, t, g = inputs(rows, dim, vocab, abi.F32)
    s = hb.HipStream()
    X, W, T, G = (Tensor.from_f32_on_stream(a, np.shape(a), s) for a in (x, w, t.astype(np.float32), g))
    _, grads = value_and_grad(X.linear_cross_entropy(W, T).mul(G).sum_all(), [X, W])
    eval_all(grads)
    for name, a, (v, b) in zip(("dx", "dw"), grads, bounds(x, w, t, g, abi.F32)):
        R.check(a.to_numpy().astype(np.float64), v, b, name)
    s.close()


@pytest.mark.parametrize("rows", [8, 16, 30, 64, 128])
@pytest.mark.parametrize("dim", [768, 2000, 4001])
def test_long_rows_are_not_summed_in_one_chain(rows, dim):
    """f32 logits of few rows are as exact, in the mean square, as sums of 48 columns
    that are added up: half as far off again, for other orders, and u / 2 for lse's own
    rounding, exponentials and logarithm."""
    x, w, t, g = T.inputs(rows, dim, 600, abi.F32, ignored=0.0)
    lse = run(x, w, t, g, abi.F32)[1]
    z = np.zeros((rows, 600), np.float32)
    for k in range(0, dim, 48):
        part = np.zeros_like(z)
        for j in range(k, min(k + 48, dim)):
            part += x[:, j:j + 1] * w[:, j]
        z += part
    exact = lse_of(x.astype(np.float64) @ w.astype(np.float64).T)
    rms = lambda a: np.sqrt((((a - exact) / exact) ** 2).mean())
    print(f"{rows} rows of {dim}: {rms(lse) / U:.2f} u, in pieces {rms(lse_of(z.astype(np.float64))) / U:.2f} u", flush=True)
    assert rms(lse) <= 1.5 * rms(lse_of(z.astype(np.float64))) + U / 2


def lse_of(z):
    m = z.max(1)
    return np.log(np.exp(z - m[:, None]).sum(1)) + m
