"""Attention of packed sequences with grouped heads and its gradients against 64
bits, within the bounds of attention_ref.py."""
import numpy as np
import pytest

import attention_ref as A
import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

LEFT = 7.0  # what results hold before the call


@pytest.fixture(params=[(-1, 0), (0, 0), (1, 0), (0, 5)], ids=["by size", "many rows", "few rows", "shares"])
def plan(request):
    """The kernels that larger or smaller calls take, at these sizes."""
    abi.load_library().mlxhip_debug_attention_plan(*request.param)
    yield
    abi.load_library().mlxhip_debug_attention_plan(-1, 0)


def inputs(tokens, heads, kv_heads, dim, dt, seed=1, std=1.0):
    return [R.rounded(synth.normal(seed + i, (tokens, h, dim), std=std), dt)
            for i, h in enumerate((heads, kv_heads, kv_heads, heads))]


class Call:
    """q, k and v side by side in one array's rows, as are the gradients; guards around all."""

    def __init__(self, q, k, v, do, starts, dt, extra=0):
        self.n, self.h, self.d = q.shape
        self.kv, self.dt, self.starts = k.shape[1], dt, np.asarray(starts, np.int32)
        self.row = (self.h + 2 * self.kv) * self.d + extra
        self.o_row = self.h * self.d + extra
        rows = np.full((self.n, self.row), LEFT, np.float32)
        for at, t in zip(self.columns(), (q, k, v)):
            rows[:, at] = t.reshape(self.n, -1)
        g = np.full((self.n, self.o_row), LEFT, np.float32)
        g[:, :self.h * self.d] = do.reshape(self.n, -1)
        self.QKV, self.G, self.S = R.Dev(rows, dt), R.Dev(g, dt), R.Dev(self.starts, abi.I32)
        self.O, self.D = R.Dev(np.full(g.shape, LEFT), dt), R.Dev(np.full(rows.shape, LEFT), dt)
        self.L = R.Dev(np.full((self.n, self.h), LEFT), abi.F32)

    def columns(self):
        h, kv, d = self.h, self.kv, self.d
        return slice(0, h * d), slice(h * d, (h + kv) * d), slice((h + kv) * d, (h + 2 * kv) * d)

    def args(self, scale, causal, stream):
        return (len(self.starts) - 1, self.n, self.h, self.kv, self.d, self.row, self.row, self.o_row, scale, causal, stream)

    def parts(self, dev):
        size = 4 if self.dt == abi.F32 else 2
        return [dev.ptr + c.start * size for c in self.columns()]

    def forward(self, scale, causal, stream=None, lse=True):
        hb.packed_attention(self.dt, *self.parts(self.QKV), self.S.ptr, self.O.ptr, self.L.ptr if lse else None,
                            *self.args(scale, causal, stream))

    def backward(self, scale, causal, stream=None):
        hb.packed_attention_vjp(self.dt, *self.parts(self.QKV), self.O.ptr, self.G.ptr, self.L.ptr, self.S.ptr,
                                *self.parts(self.D), *self.args(scale, causal, stream))

    def results(self):
        o, d = self.O.get(), self.D.get()
        assert (o[:, self.h * self.d:] == LEFT).all() and (d[:, (self.h + 2 * self.kv) * self.d:] == LEFT).all()
        grads = [d[:, c].reshape(self.n, -1, self.d) for c in self.columns()]
        return [o[:, :self.h * self.d].reshape(self.n, self.h, self.d), self.L.get()] + grads


def compare(q, k, v, do, starts, scale, causal, dt, extra=0, stream=None):
    c = Call(q, k, v, do, starts, dt, extra)
    c.forward(scale, causal, stream)
    c.backward(scale, causal, stream)
    hb.synchronize(stream)
    o, lse, *grads = c.results()
    wo, eo, wl, el = A.packed(q, k, v, starts, scale, causal, dt)
    rest = A.same_where(o, wo, eo, "o")
    assert (o[rest] == LEFT).all()
    rest = A.same_where(lse, wl, el, "lse")
    assert (lse[rest] == LEFT).all()
    for name, got, (want, bound) in zip(("dq", "dk", "dv"), grads, A.packed_vjp(q, k, v, do, starts, scale, causal, dt)):
        rest = A.same_where(got, want, bound, name)
        assert (got[rest] == LEFT).all(), name


# tokens, heads, kv_heads, dim, starts
CASES = [(1, 1, 1, 8, [0, 1]), (2, 2, 1, 64, [0, 1, 2]), (33, 3, 3, 16, [0, 33]), (64, 4, 1, 128, [0, 64]),
         (65, 6, 2, 80, [0, 1, 65]), (129, 8, 8, 64, [0, 63, 63, 129]), (200, 5, 1, 120, [0, 70, 199]),
         (300, 9, 3, 72, [5, 135, 136, 290]), (257, 16, 2, 128, [0, 257]), (515, 2, 2, 128, [0, 130, 515]),
         (90, 7, 7, 24, [0, 0, 0, 90]), (400, 16, 8, 40, [0, 31, 95, 223, 400])]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("tokens,heads,kv,dim,starts", CASES)
def test_matches_64_bits(tokens, heads, kv, dim, starts, causal, dt, plan):
    print(f"packed {tokens} {heads}/{kv} {dim} {starts} causal {causal} {R.NAMES[dt]}", flush=True)
    compare(*inputs(tokens, heads, kv, dim, dt, seed=dim), starts, dim ** -0.5, causal, dt)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 2.0 ** -40])
def test_other_scales(scale, dt, plan):
    compare(*inputs(70, 4, 2, 32, dt), [0, 20, 70], scale, True, dt)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_rows_apart(dt, plan):
    compare(*inputs(100, 4, 2, 48, dt), [0, 37, 100], 0.2, True, dt, extra=24)


@pytest.mark.parametrize("dt", [abi.F32, abi.BF16], ids=R.NAMES.get)
def test_rows_as_far_apart_as_may_be(dt):
    """2^20 elements, and heads that end inside a tile's row: what is past them stays zeros."""
    compare(*inputs(70, 1, 1, 40, dt), [0, 70], 0.2, True, dt, extra=(1 << 20) - 120)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_certain_rows(dt, plan):
    """Scores of +-100: probabilities of 1 and 0, a maximum that moves late and far."""
    q, k, v, do = inputs(150, 2, 1, 64, dt)
    q = R.rounded(4 * q, dt)
    k = R.rounded(k * np.linspace(0.1, 4, 150, dtype=np.float32)[:, None, None], dt)
    compare(q, k, v, do, [0, 150], 0.35, True, dt)


@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -12, 2.0 ** 8])
def test_f16_gradients_keep_their_digits(size, plan):
    """Cotangents whose dS lies below or far above f16's normal range; q, k and v so that
    the results are in it."""
    q, k, v, do = inputs(260, 4, 2, 64, abi.F16)
    if size < 1:
        q, k = (R.rounded(t * 2.0 ** 5, abi.F16) for t in (q, k))
    compare(q, k, v, R.rounded(do * size, abi.F16), [0, 3, 260], 2.0 ** -13 if size < 1 else 0.125, True, abi.F16)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("dim", [64, 128])
def test_non_finite_values_stay_with_those_that_see_them(dim, dt, plan):
    """Of another sequence, of keys that a causal row does not see, of tokens of no
    sequence: rows that see none are as without them."""
    q, k, v, do = inputs(300, 4, 2, dim, dt)
    starts = [0, 100, 290]
    clean = Call(q, k, v, do, starts, dt)
    clean.forward(0.1, True)
    bad = [t.copy() for t in (k, v)]
    for t, val in zip(bad, (np.nan, np.inf)):
        t[140, 1], t[295] = val, val
        t[231, 0, 3] = -np.inf if val == np.inf else val
    c = Call(q, *bad, do, starts, dt)
    c.forward(0.1, True)
    hb.synchronize()
    (o, lse, *_), (want, wl, *_) = c.results(), clean.results()
    sees = np.zeros((300, 4), bool)
    sees[140:290, 2:] = True
    sees[231:290, :2] = True
    np.testing.assert_array_equal(o[~sees], want[~sees])
    np.testing.assert_array_equal(lse[~sees], wl[~sees])
    assert (~np.isfinite(o[140:290, 2:])).any(2).all() and (~np.isfinite(o[231:290, :2, 3])).all()


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_non_finite_values_that_carry_no_weight(dt, plan):
    """0 times NaN: of 32 keys whose scores lie 400 below the others', one in v."""
    q, k, v, do = inputs(100, 2, 1, 16, dt)
    q[:], k[:] = 10.0, 0.0
    k[:32, :, 0] = -40.0
    v[5, 0, 3] = np.nan
    c = Call(q, k, v, do, [0, 100], dt)
    c.forward(1.0, True)
    hb.synchronize()
    o = c.results()[0]
    assert np.isnan(o[5:, :, 3]).all() and np.isfinite(o[:5]).all()
    assert np.isfinite(np.delete(o, 3, axis=2)).all()


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_rows_without_any_score(dt, plan):
    """Scores of -inf everywhere a row sees: 0/0, as the formula says."""
    q, k, v, do = inputs(40, 1, 1, 16, dt)
    q, k = np.abs(q) + 1, k.copy()
    q = R.rounded(q, dt)
    k[:4] = -np.inf
    c = Call(q, k, v, do, [0, 40], dt)
    c.forward(1.0, True)
    hb.synchronize()
    o = c.results()[0]
    assert np.isnan(o[:4]).all() and np.isfinite(o[4:]).all()
    want, bound, *_ = A.attend(*(t[4:, 0].astype(np.float64) for t in (q, k, v)), 0, 1.0, True, dt)
    R.check(o[4:, 0], want, bound + R.U * 8 * np.abs(want), "the others")


def test_gradients_against_differences(plan):
    tokens, starts, scale = 50, [0, 17, 50], 0.3
    q, k, v, do = inputs(tokens, 4, 2, 16, abi.F32)
    c = Call(q, k, v, do, starts, abi.F32)
    c.forward(scale, True)
    c.backward(scale, True)
    hb.synchronize()
    grads = c.results()[2:]
    h = 2.0 ** -6
    for i, name in enumerate("qkv"):
        d = synth.normal(40 + i, (q, k, v)[i].shape)
        out = []
        for s in (h, -h):
            t = [q, k, v]
            t[i] = (t[i] + np.float32(s) * d).astype(np.float32)
            w, *_ = A.packed(*t, starts, scale, True, abi.F32)
            out.append((w * do).sum())
        slope, want = (out[0] - out[1]) / (2 * h), (grads[i] * d).sum()
        # A central difference is off by h^2 / 6 of the third derivative; sums of 50 * 64 terms of about 1.
        assert abs(slope - want) <= h * h * 60 + 1e-3, (name, slope, want)


def test_no_tokens_and_no_sequences():
    hb.packed_attention(abi.BF16, 0, 0, 0, 0, 0, None, 0, 0, 4, 2, 64, 256, 128, 256, 0.1)
    hb.packed_attention(abi.F32, 0, 0, 0, 0, 0, None, 3, 0, 4, 2, 64, 256, 128, 256, 0.1)
    c = Call(*inputs(5, 2, 1, 16, abi.F32), [2, 2, 2], abi.F32)
    c.forward(1.0, True)
    c.backward(1.0, True)
    hb.synchronize()
    assert all((t == LEFT).all() for t in c.results())


@pytest.mark.parametrize("starts", [[0, 40, 20, 64], [-5, 30, 1000], [64, 0, 0], [2**31 - 1, -2**31, 10]])
def test_any_starts_stay_in_bounds(starts, plan):
    """Not ascending, or outside: no values are promised, nothing outside the arrays is touched."""
    c = Call(*inputs(64, 4, 2, 32, abi.BF16), starts, abi.BF16)
    c.forward(0.2, True)
    c.backward(0.2, True)
    hb.synchronize()
    c.results()


def test_many_short_sequences(plan):
    lengths = (synth.uniform01(3, 150) * 6).astype(int)
    starts = np.concatenate([[0], np.cumsum(lengths)])
    compare(*inputs(int(starts[-1]) + 3, 4, 2, 16, abi.F32), starts, 0.25, True, abi.F32)


@pytest.mark.parametrize("n,most,first", [(5000, 3, 0), (5000, 2, 9), (130, 90, 3), (64, 50, 0), (65, 50, 1)])
def test_thousands_of_sequences(n, most, first, plan):
    """More than 64 times 64, empty ones among them, tokens in front of and behind them."""
    lengths = (synth.uniform01(4, n) * most).astype(int)
    starts = first + np.concatenate([[0], np.cumsum(lengths)])
    compare(*inputs(int(starts[-1]) + 2, 2, 1, 8, abi.F32), starts, 0.25, True, abi.F32)


@pytest.mark.parametrize("dt", [abi.F32, abi.F16], ids=R.NAMES.get)
def test_same_bits_every_time_and_replayed(dt, plan):
    data, starts = inputs(333, 8, 2, 64, dt), [0, 100, 333]
    def fresh():
        return Call(*data, starts, dt)
    one = fresh()
    one.forward(0.125, True)
    one.backward(0.125, True)
    hb.synchronize()
    want = one.results()
    s = hb.create_stream()
    try:
        a, b = fresh(), fresh()
        a.forward(0.125, True, s)
        a.backward(0.125, True, s)
        with hb.Graph(s) as g:
            b.forward(0.125, True, s)
            b.backward(0.125, True, s)
        for _ in range(3):
            g.launch()
            one.forward(0.125, True)  # eager work beside the replay
            hb.synchronize(s)
            hb.synchronize()
            for got in (a.results(), b.results(), one.results()):
                for x, y in zip(got, want):
                    np.testing.assert_array_equal(x, y)
        g.close()
    finally:
        hb.destroy_stream(s)


def test_offsets_beyond_32_bits():
    """Rows 2 MiB apart: the last of 2200 tokens lies 4.6 GB behind the first."""
    tokens, row, dt = 2200, 1 << 20, abi.BF16
    q, k, v, do = inputs(tokens, 2, 1, 16, dt)
    starts = [0, 2150, 2200]
    buf = hb.DeviceBuffer(tokens * row * 2)
    part = np.concatenate([t.reshape(tokens, -1) for t in (q, k, v)], 1)
    bits = synth.bf16_bits(part).reshape(tokens, -1)
    for t in range(tokens):
        buf.upload(bits[t], t * row * 2)
    S, O, L = R.Dev(starts, abi.I32), R.Dev(dt=dt, shape=(tokens, 32)), R.Dev(dt=abi.F32, shape=(tokens, 2))
    G = R.Dev(do, dt)
    args = (2, tokens, 2, 1, 16, row, row, 32, 0.25, True)
    at = [buf.ptr + 2 * c for c in (0, 32, 48)]
    hb.packed_attention(dt, *at, S.ptr, O.ptr, L.ptr, *args)
    grads = [buf.ptr + 2 * c for c in (64, 96, 112)]
    hb.packed_attention_vjp(dt, *at, O.ptr, G.ptr, L.ptr, S.ptr, *grads, *args)
    hb.synchronize()
    i = slice(2150, 2200)
    got = np.stack([buf.download(np.uint16, 64, t * row * 2 + 128) for t in range(2150, 2200)])
    got = synth.bf16_to_f32(got).astype(np.float64)
    wo, eo, wl, el = A.packed(q[i], k[i], v[i], [0, 50], 0.25, True, dt)
    R.check(O.get().reshape(tokens, 2, 16)[i], wo, eo, "o")
    wants = A.packed_vjp(q[i], k[i], v[i], do[i], [0, 50], 0.25, True, dt)
    for name, cols, (want, bound) in zip(("dq", "dk", "dv"), (slice(0, 32), slice(32, 48), slice(48, 64)), wants):
        R.check(got[:, cols].reshape(want.shape), want, bound, name)
    buf.free()


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_a_training_step_of_rotated_heads(dt):
    """Rotary positions that start anew with each sequence, attention, and back: queries
    and keys turned in place in the projection's rows, their gradients turned back."""
    from test_gpu_rope_rows import frequencies
    q, k, v, do = inputs(120, 4, 2, 32, dt)
    starts, f = [0, 50, 120], frequencies(24)
    pos = np.concatenate([np.arange(50), np.arange(70)]).astype(np.int32)
    c = Call(q, k, v, do, starts, dt)
    P, F = R.Dev(pos, abi.I32), hb.DeviceBuffer.from_array(f)
    turn = (120, 6, 32, 24, c.row, c.row, False)  # q's and k's heads lie side by side
    hb.rope_rows(dt, c.QKV.ptr, P.ptr, F, c.QKV.ptr, *turn)
    c.forward(0.2, True)
    c.backward(0.2, True)
    hb.rope_vjp_rows(dt, c.D.ptr, P.ptr, F, c.D.ptr, *turn)
    hb.synchronize()
    o, lse, dq, dk, dv = c.results()
    tq, tk = (R.rounded(A.rope(t, pos, f, 24, False, 1.0, dt)[0].astype(np.float32), dt) for t in (q, k))
    wo, eo, _, _ = A.packed(tq, tk, v, starts, 0.2, True, dt)
    wants = A.packed_vjp(tq, tk, v, do, starts, 0.2, True, dt)
    # A value turned in f32 may round to the other neighbour, a step of 2 HALF of it: scores move by 4 HALF of
    # their terms' magnitudes, and dS, a product of two such, by as much of itself.
    z = 0.2 * 4 * R.HALF[dt] * (np.abs(tq).sum(2).max() * np.abs(tk).max())
    R.check(o, wo, eo + 2 * z * np.abs(v).max(), "o")
    for name, got, (want, bound), turned in zip(("dq", "dk", "dv"), (dq, dk, dv), wants, (True, True, False)):
        size = np.abs(want).max() + 0.2 * np.abs(do).sum(2).max() * np.abs(v).max() * (np.abs(tq).max() + np.abs(tk).max())
        bound = bound + 4 * z * size * (1 if turned else 2)
        if turned:
            want, e = A.rope(want, pos, f, 24, False, 1.0, dt, -1.0)
            bound = e + 2 * bound.max(2, keepdims=True)
        R.check(got, want, bound, name)
