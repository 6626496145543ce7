"""Values of v next to the largest numbers of f32 and bf16: sums of p v that pass them where
the result, divided by the sum of p, does not."""
import numpy as np
import pytest

import attention_ref as A
import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb
from test_gpu_packed_attention import Call, inputs, plan  # noqa: F401 (a fixture)
from test_gpu_paged_attention import Cache

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

TYPES = [abi.F32, abi.BF16]


def large(shape, dt, seed=7):
    """2^126 to 1.9 times that."""
    return R.rounded(((1 + 0.9 * synth.uniform01(seed, int(np.prod(shape))).reshape(shape)) * 2.0 ** 126).astype(np.float32), dt)


@pytest.mark.parametrize("dt", TYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("dim", [32, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_packed(causal, dim, dt, plan):  # noqa: F811
    """Large values from the 150th token of one K/V head on, in every other place of a row: rows
    that see none of them are as without them, bit for bit."""
    q, k, v, do = inputs(400, 4, 2, dim, dt)
    starts = [0, 300, 390]
    clean = Call(q, k, v, do, starts, dt)
    clean.forward(0.1, causal)
    v[150:, 1, ::2] = large(v[150:, 1, ::2].shape, dt)
    c = Call(q, k, v, do, starts, dt)
    c.forward(0.1, causal)
    hb.synchronize()
    (o, lse, *_), (was, wl, *_) = c.results(), clean.results()
    want, eo, wlse, el = A.packed(q, k, v, starts, 0.1, causal, dt)
    A.same_where(o, want, eo, "o")
    A.same_where(lse, wlse, el, "lse")
    sees = np.zeros((400, 4), bool)
    sees[150 if causal else 0:390, 2:] = True
    np.testing.assert_array_equal(o[~sees], was[~sees])
    np.testing.assert_array_equal(lse, wl)


@pytest.mark.parametrize("dt", TYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("lens", [[300, 90], [5000, 700]])
def test_paged(lens, new, dt):
    """Whole walks, and parts of which some hold large values."""
    c = Cache(lens, [new, 1], 8, 2, 64, 16, dt)
    c.v[0][70:200, :, 1::2] = large(c.v[0][70:200, :, 1::2].shape, dt)
    c.v[1][:, 0] = large(c.v[1][:, 0].shape, dt, 8)
    R.check(c.attend(0.1), *c.want(0.1), "o")


@pytest.mark.parametrize("dt", TYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("lens,apart", [(200, 32), (2000, 256)])
def test_sums_that_pass_it_only_when_joined(lens, apart, new, dt):
    """One key that counts in each wave's tile, or in each part: every sum is finite, that of
    two of them is not."""
    c = Cache([lens], [new], 4, 1, 16, 16, dt)
    c.q[:], c.k[0][:] = 4.0, 0.0
    c.k[0][5::apart] = 4.0
    c.v[0][5::apart] = R.rounded(np.full(c.v[0][5::apart].shape, 1.5 * 2.0 ** 127, np.float32), dt)
    R.check(c.attend(1.0), *c.want(1.0), "o")


@pytest.mark.parametrize("dt", TYPES, ids=R.NAMES.get)
def test_non_finite_values_beside_small_ones(dt, plan):  # noqa: F811
    """A row that sees no value that is not finite keeps the digits of values down to 2^-100."""
    q, k, v, do = inputs(100, 2, 1, 32, dt)
    v = (v * np.float32(2.0 ** -100)).astype(np.float32)
    clean = Call(q, k, v, do, [0, 100], dt)
    clean.forward(0.2, True)
    v[60] = np.inf
    c = Call(q, k, v, do, [0, 100], dt)
    c.forward(0.2, True)
    hb.synchronize()
    o, was = c.results()[0], clean.results()[0]
    np.testing.assert_array_equal(o[:60], was[:60])
    assert (~np.isfinite(o[60:])).all()
