"""Rotary positions of rows and their gradient against 64 bits."""
import numpy as np
import pytest

import attention_ref as A
import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


def frequencies(rotary, base=10000.0, factor=1.0, low=0.0, high=0.0, original=0):
    f = base ** (-2.0 * np.arange(rotary // 2) / rotary)
    if factor == 1.0:
        return f
    keep = np.clip((original * f / (2 * np.pi) - low) / (high - low), 0, 1) if original else 0.0
    return f * (keep + (1 - keep) / factor)


def turned(x, positions, freqs, rotary, interleaved, dt, vjp=False, magnitude=1.0, stride=0, offset=0, stream=None,
           in_place=False):
    """The kernel's result for x [tokens, heads, dim]; with a stride, what lies between rows must stay."""
    n, h, d = x.shape
    stride = stride or h * d
    host = np.full((n, stride), 7.0, np.float32)
    host[:, :h * d] = x.reshape(n, -1)
    X, P = R.Dev(host, dt, offset), R.Dev(positions, abi.I32)
    F = hb.DeviceBuffer.from_array(np.asarray(freqs, np.float64))
    Y = X if in_place else R.Dev(np.full((n, stride), 7.0), dt, offset)
    f = hb.rope_vjp_rows if vjp else hb.rope_rows
    f(dt, X.ptr, P.ptr, F, Y.ptr, n, h, d, rotary, stride, stride, interleaved, magnitude, stream)
    hb.synchronize(stream)
    y = Y.get()
    assert (y[:, h * d:] == 7.0).all()
    return y[:, :h * d].reshape(n, h, d)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,dim,rotary", [(1, 1, 2, 2), (1, 12, 64, 64), (3, 5, 80, 40), (9, 3, 77, 34), (130, 40, 128, 128),
                                                (17, 1, 1024, 1024), (5, 7, 33, 2), (2, 64, 256, 250)])
def test_matches_64_bits(n, heads, dim, rotary, interleaved, dt):
    print(f"rope {n} {heads} {dim} {rotary} {R.NAMES[dt]}", flush=True)
    x = R.rounded(synth.normal(n + dim, (n, heads, dim)), dt)
    pos = (synth.uniform01(dim, n) * 200000).astype(np.int32)
    f = frequencies(rotary)
    for vjp in (False, True):
        want, bound = A.rope(x, pos, f, rotary, interleaved, 1.0, dt, -1.0 if vjp else 1.0)
        R.check(turned(x, pos, f, rotary, interleaved, dt, vjp), want, bound, f"vjp {vjp}")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary,offset", [(77, 34, 1), (64, 64, 3), (24, 18, 5)])
def test_any_alignment_strides_in_place(dim, rotary, offset, interleaved, dt):
    x = R.rounded(synth.normal(dim, (11, 3, dim)), dt)
    pos, f = np.arange(-5, 6, dtype=np.int32), frequencies(rotary)
    want, bound = A.rope(x, pos, f, rotary, interleaved, 1.25, dt)
    for in_place in (False, True):
        got = turned(x, pos, f, rotary, interleaved, dt, magnitude=1.25, stride=3 * dim + 13, offset=offset, in_place=in_place)
        R.check(got, want, bound, f"in place {in_place}")


def test_far_positions_keep_their_angles():
    pos = np.array([0, 1, 2**24 + 1, 2**30 + 12345, 2**31 - 1, -2**31], np.int32)
    x, f = synth.normal(3, (len(pos), 2, 64)), frequencies(64)
    R.check(turned(x, pos, f, 64, False, abi.F32), *A.rope(x, pos, f, 64, False, 1.0, abi.F32), "far")


@pytest.mark.parametrize("args", [(10000.0,), (500000.0, 8.0, 1.0, 4.0, 8192), (10000.0, 4.0), (1e6, 1.0, 0.0, 0.0, 4096),
                                  (10000.0, 32.0, 1.0, 1.5, 131072)], ids=str)
@pytest.mark.parametrize("rotary", [2, 34, 128, 1024])
def test_frequencies(rotary, args):
    F = hb.DeviceBuffer(rotary // 2 * 8)
    hb.rope_frequencies(F, rotary, *args)
    hb.synchronize()
    np.testing.assert_allclose(F.download(np.float64), frequencies(rotary, *args), rtol=1e-13)


def test_the_gradient_is_the_transpose():
    """sum(dy rope(x)) = sum(rope_vjp(dy) x), and against differences."""
    x, dy = synth.normal(1, (6, 3, 40)), synth.normal(2, (6, 3, 40))
    pos, f = np.arange(6, dtype=np.int32) * 1000, frequencies(24)
    y, dx = turned(x, pos, f, 24, True, abi.F32), turned(dy, pos, f, 24, True, abi.F32, vjp=True)
    mag = np.abs(dy * y).sum() + np.abs(dx * x).sum()
    assert abs((dy * y).sum() - (dx * x).sum()) <= 20 * R.U * mag
    d = synth.normal(5, x.shape)
    ahead, behind = (turned((x + s * d).astype(np.float32), pos, f, 24, True, abi.F32) for s in (0.5, -0.5))
    # Linear: a difference of any width, off by the steps' rounding.
    assert abs((dy * (ahead - behind)).sum() - (dx * d).sum()) <= 40 * R.U * (mag + np.abs(dy).sum() * 8)


def test_non_finite_values_stay_in_their_pairs():
    x = synth.normal(1, (3, 2, 16))
    x[1, 0, 3] = np.nan
    x[2, 1, 15] = np.inf
    got = turned(x, np.arange(3, dtype=np.int32), frequencies(12), 12, False, abi.F32)
    bad = ~np.isfinite(got)
    assert bad[1, 0, 3] and bad[1, 0, 9] and got[2, 1, 15] == np.inf and bad.sum() == 3


def test_nothing_to_turn():
    hb.rope_rows(abi.F32, 0, 0, 0, 0, 0, 3, 8, 8, 24, 24)
    hb.rope_rows(abi.F16, 0, 0, 0, 0, 5, 0, 8, 8, 0, 0)


@pytest.mark.parametrize("n", [5, 3000])
def test_same_bits_on_another_stream_and_replayed(n):
    x = R.rounded(synth.normal(4, (n, 6, 48)), abi.BF16)
    pos, f = np.arange(n, dtype=np.int32), frequencies(48)
    one = turned(x, pos, f, 48, False, abi.BF16)
    s = hb.create_stream()
    try:
        np.testing.assert_array_equal(one, turned(x, pos, f, 48, False, abi.BF16, stream=s))
        X, P, Y = R.Dev(x, abi.BF16), R.Dev(pos, abi.I32), R.Dev(dt=abi.BF16, shape=x.shape)
        F = hb.DeviceBuffer(24 * 8)
        with hb.Graph(s) as g:
            hb.rope_frequencies(F, 48, 10000.0, stream=s)
            hb.rope_rows(abi.BF16, X.ptr, P.ptr, F, Y.ptr, n, 6, 48, 48, 288, 288, False, 1.0, s)
        for _ in range(3):
            g.launch()
            hb.synchronize(s)
            np.testing.assert_array_equal(one, Y.get())
        g.close()
    finally:
        hb.destroy_stream(s)
