"""Forms of the rotary and packed calls that only large or forward-only work takes: rotary
rows of 64 MiB and more, which are stored past the caches, and attention without lse."""
import numpy as np
import pytest

import attention_ref as A
import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb
from test_gpu_packed_attention import LEFT, Call, inputs, plan  # noqa: F401 (a fixture)
from test_gpu_rope_rows import frequencies, turned

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_large_rotary_rows(in_place, interleaved, dt):
    """Odd heads of 77, rows an odd number of elements apart from an odd element on: the same rows
    over and over, each time with the bits that a small call gives them."""
    n, heads, dim, rotary = 499, 9, 77, 34
    times = -(-(1 << 26) // (n * heads * dim * (4 if dt == abi.F32 else 2)))
    print(f"rope {n * times} x {heads} x {dim} {R.NAMES[dt]}", flush=True)
    x = R.rounded(synth.normal(3, (n, heads, dim)), dt)
    pos, f = (synth.uniform01(4, n) * 200000).astype(np.int32), frequencies(rotary)
    how = dict(stride=heads * dim + 14, offset=1, in_place=in_place)
    for vjp in (False, True):
        small = turned(x, pos, f, rotary, interleaved, dt, vjp, **how)
        R.check(small, *A.rope(x, pos, f, rotary, interleaved, 1.0, dt, -1.0 if vjp else 1.0), f"vjp {vjp}")
        got = turned(np.tile(x, (times, 1, 1)), np.tile(pos, times), f, rotary, interleaved, dt, vjp, **how)
        np.testing.assert_array_equal(got.reshape(times, n, heads, dim), np.broadcast_to(small, (times, n, heads, dim)))


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_without_lse(causal, dt, plan):  # noqa: F811
    data, starts = inputs(300, 6, 2, 72, dt), [2, 130, 131, 290]
    a, b = Call(*data, starts, dt), Call(*data, starts, dt)
    a.forward(0.12, causal)
    b.forward(0.12, causal, lse=False)
    hb.synchronize()
    (o, lse, *_), (alone, none, *_) = a.results(), b.results()
    assert (lse[2:290] != LEFT).all() and (none == LEFT).all()
    np.testing.assert_array_equal(o, alone)
