"""Targets of the lazy linear cross entropy that are no whole number of the
vocabulary: they take their rows out of the loss, its mean and the gradients."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, nn, synth
from oxidizedmlx_amd import backend as hb
from oxidizedmlx_amd.tensor import Tensor, eval_all, value_and_grad

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

VOCAB = 333
ODD = [2.5, VOCAB - 0.5, 0.25, -0.5, 1e-30, np.nextafter(np.float32(7), np.float32(8)), 2.0 ** 24, np.nan, -np.inf]


def const(a, s):
    return Tensor.from_f32_on_stream(a, np.shape(a), s)


@pytest.fixture(params=[False, True], ids=["sync", "async"])
def stream(request):
    s = hb.HipStream(async_eval=request.param)
    yield s
    s.close()


def inputs(rows):
    x, w = synth.normal(1, (rows, 48)), synth.normal(2, (VOCAB, 48), 0.0, 0.3)
    t = np.floor(synth.uniform01(3, rows) * VOCAB).astype(np.float32)
    t[:len(ODD)] = ODD
    whole = np.where(np.arange(rows) < len(ODD), -1, np.nan_to_num(t)).astype(np.int32)
    return x, w, t, whole


@pytest.mark.parametrize("rows", [12, 70, 200])
def test_a_fraction_is_no_target(stream, rows):
    x, w, t, whole = inputs(rows)
    g = synth.normal(4, (rows,))
    X, W = const(x, stream), const(w, stream)
    loss = X.linear_cross_entropy(W, const(t, stream))
    _, grads = value_and_grad(loss.mul(const(g, stream)).sum_all(), [X, W])
    eval_all([loss, *grads])
    R.check(loss.to_numpy().astype(np.float64), *R.cross_entropy(x, w, whole, abi.F32)[0], "loss")
    # lse comes from the loss: twice the bound, as where it is given whole targets.
    for name, a, (v, b) in zip(("dx", "dw"), grads, R.cross_entropy_vjp(x, w, whole, g, abi.F32)):
        R.check(a.to_numpy().astype(np.float64), v, 2 * b, name)


@pytest.mark.parametrize("rows", [12, 70, 200])
def test_a_fraction_does_not_count_in_the_mean(stream, rows):
    """The same bits as with -1 in its place."""
    x, w, t, whole = inputs(rows)
    seen = []
    for targets in (t.astype(np.float64), whole):
        X, W = const(x, stream), const(w, stream)
        loss, grads = value_and_grad(nn.LinearCrossEntropy(W)(X, targets), [X, W])
        eval_all([loss, *grads])
        seen.append([a.to_numpy() for a in (loss, *grads)])
    for a, b in zip(*seen):
        np.testing.assert_array_equal(a, b)
