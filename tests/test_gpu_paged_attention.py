"""A cache in pages: append with rotary positions, and attention of new tokens over
it, against 64 bits within the bounds of attention_ref.py."""
import numpy as np
import pytest

import attention_ref as A
import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

LEFT = 7.0


class Cache:
    """Pages of NaN, sequences of `lens` positions, `new` of them this step's."""

    def __init__(self, lens, new, heads, kv_heads, dim, page, dt, seed=1, width=None):
        self.lens, self.new = np.asarray(lens, np.int32), np.asarray(new)
        self.starts = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.tokens, self.h, self.kv, self.d, self.page, self.dt = int(self.starts[-1]), heads, kv_heads, dim, page, dt
        rng = np.random.default_rng(seed)
        per = [-(-max(int(n), 0) // page) for n in lens]
        self.pages, self.width = sum(per) + 2, width or max(max(per), 1)
        self.table = A.pages_of(lens, page, max(self.width, max(per)), self.pages, rng)[:, :self.width]
        self.k = [R.rounded(synth.normal(seed + 10 + i, (max(int(n), 0), kv_heads, dim)), dt) for i, n in enumerate(lens)]
        self.v = [R.rounded(synth.normal(seed + 1010 + i, (max(int(n), 0), kv_heads, dim)), dt) for i, n in enumerate(lens)]
        self.q = R.rounded(synth.normal(seed, (self.tokens, heads, dim)), dt)

    def filled(self, rows, fill=np.nan):
        """The pages holding rows[s][p] at the table's places."""
        out = np.full((self.pages, self.kv, self.page, self.d), fill, np.float32)
        for s, r in enumerate(rows):
            for p in range(min(len(r), self.width * self.page)):
                out[self.table[s, p // self.page], :, p % self.page] = r[p]
        return out

    def attend(self, scale, stream=None, k=None, v=None, extra=0, q=None):
        K, V = R.Dev(self.filled(k or self.k), self.dt), R.Dev(self.filled(v or self.v), self.dt)
        row = self.h * self.d + extra
        host = np.full((self.tokens + 2, row), LEFT, np.float32)  # two rows behind the last sequence
        host[:self.tokens, :self.h * self.d] = (self.q if q is None else q).reshape(self.tokens, -1)
        Q, O = R.Dev(host, self.dt), R.Dev(np.full(host.shape, LEFT), self.dt)
        S, N, T = (R.Dev(t, abi.I32) for t in (self.starts, self.lens, self.table))
        args = (self.dt, Q.ptr, K.ptr, V.ptr, S.ptr, N.ptr, T.ptr, O.ptr, len(self.lens), self.tokens + 2, self.h, self.kv,
                self.d, row, row, self.pages, self.page, self.width, scale, stream)
        hb.paged_attention(*args)
        hb.synchronize(stream)
        o = O.get()
        assert (o[self.tokens:] == LEFT).all() and (o[:, self.h * self.d:] == LEFT).all()
        return o[:self.tokens, :self.h * self.d].reshape(self.tokens, self.h, self.d)

    def want(self, scale, q=None):
        q = np.asarray(self.q if q is None else q, np.float64)
        o, e = np.zeros(q.shape), np.zeros(q.shape)
        for s, (n, m) in enumerate(zip(self.lens, self.new)):
            at, room = self.starts[s], self.width * self.page
            k, v = (np.asarray(t[s][:room], np.float64) for t in (self.k, self.v))
            for h in range(self.h if m else 0):
                g = h * self.kv // self.h
                o[at:at + m, h], e[at:at + m, h], *_ = A.attend(q[at:at + m, h], k[:, g], v[:, g], int(n) - int(m), scale, True,
                                                               self.dt)
        return o, e


CASES = [  # lens, new, heads, kv_heads, dim, page
    ([1], [1], 1, 1, 8, 16), ([17, 1, 300], [1, 1, 1], 4, 1, 64, 16), ([144] * 8, [1] * 8, 12, 12, 64, 16),
    ([1000, 33, 16, 257], [1, 1, 1, 1], 8, 2, 128, 32), ([40, 500], [7, 1], 6, 2, 80, 64), ([600], [200], 4, 2, 128, 16),
    ([130, 0, 64, 70], [130, 0, 64, 3], 16, 2, 72, 128), ([2100, 5], [3, 5], 32, 1, 40, 256), ([90, 20], [33, 20], 5, 5, 120, 16),
    ([513, 512, 511], [1, 2, 3], 2, 1, 96, 512), ([3000], [1], 40, 1, 16, 16)]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("lens,new,heads,kv,dim,page", CASES)
def test_matches_64_bits(lens, new, heads, kv, dim, page, dt):
    print(f"paged {lens} {new} {heads}/{kv} {dim} page {page} {R.NAMES[dt]}", flush=True)
    c = Cache(lens, new, heads, kv, dim, page, dt)
    R.check(c.attend(dim ** -0.5), *c.want(dim ** -0.5), "o")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("new", [1, 40])
def test_wide_tables_split_their_keys(new, dt):
    """Room for far more positions than the sequences have: as many parts as their keys are worth."""
    c = Cache([5000, 255, 256, 257], [new] * 4, 8, 2, 64, 16, dt, width=4000)
    R.check(c.attend(0.2, extra=8), *c.want(0.2), "o")
    c.q = R.rounded(-8 * c.q, dt)  # certain rows: parts whose maxima lie far apart
    R.check(c.attend(0.2), *c.want(0.2), "certain")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("new", [[5, 3, 1], [60, 40, 1]])
def test_tokens_that_see_nothing_are_zeros(new, dt):
    """More new tokens than positions, a negative length, none."""
    c = Cache([2, 0, -4], new, 4, 2, 32, 16, dt)
    got = c.attend(0.3)
    want, bound = c.want(0.3)
    assert (want[:new[0] - 2] == 0).all() and (want[new[0]:] == 0).all()
    R.check(got, want, bound, "o")


def test_lengths_beyond_the_table_are_cut():
    c = Cache([100, 40], [3, 2], 4, 2, 32, 16, abi.F32, width=4)
    R.check(c.attend(0.3), *c.want(0.3), "o")


@pytest.mark.parametrize("new", [1, 50])
def test_bad_pages_read_as_zeros(new):
    c = Cache([400, 90], [new, 1], 4, 2, 64, 16, abi.BF16)
    for s, p, page in ((0, 3, -1), (0, 9, c.pages), (1, 0, 2**31 - 1), (1, 5, -2**31)):
        at = c.table[s, p]
        c.k[s][16 * p:16 * p + 16] = 0
        c.v[s][16 * p:16 * p + 16] = 0
        c.table[s, p] = page
    wanted = c.want(0.2)
    for t in (c.k, c.v):  # the places that cannot be stored
        t[0], t[1] = t[0].copy(), t[1].copy()
    keep = c.table.copy()
    c.filled = lambda rows, table=keep: _skipping(c, rows, table)
    R.check(c.attend(0.2), *wanted, "o")


def _skipping(c, rows, table):
    out = np.full((c.pages, c.kv, c.page, c.d), np.nan, np.float32)
    for s, r in enumerate(rows):
        for p in range(len(r)):
            page = table[s, p // c.page]
            if 0 <= page < c.pages:
                out[page, :, p % c.page] = r[p]
    return out


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("lens", [[100], [2000]])
def test_non_finite_values_that_carry_no_weight(lens, new):
    """0 times NaN: of 32 positions whose scores lie 400 below the others', one in v."""
    c = Cache(lens, [new], 2, 1, 16, 16, abi.BF16)
    c.q[:], c.k[0][:] = 10.0, 0.0
    c.k[0][:32, :, 0] = -40.0
    c.v[0][5, 0, 3] = np.nan
    o = c.attend(1.0)
    assert np.isnan(o[:, :, 3]).all() and np.isfinite(np.delete(o, 3, axis=2)).all()


def test_two_sequences_share_pages():
    c = Cache([64, 64], [1, 1], 4, 2, 64, 16, abi.F16)
    c.table[1, :3] = c.table[0, :3]
    for t in (c.k, c.v):
        t[1][:48] = t[0][:48]
    R.check(c.attend(0.2), *c.want(0.2), "o")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("rotary,interleaved", [(0, False), (64, False), (40, True), (18, False)])
@pytest.mark.parametrize("page", [16, 64])
def test_append(page, rotary, interleaved, dt):
    from test_gpu_rope_rows import frequencies
    new, lens = [3, 0, 70, 1], [3, 20, 150, 41]
    c = Cache(lens, new, 4, 3, 64, page, dt)
    row = 2 * 3 * 64
    kv = R.rounded(synth.normal(77, (c.tokens + 2, 2, 3, 64)), dt)
    before = [[r[:n - m] for r, n, m in zip(t, lens, new)] for t in (c.k, c.v)]
    KV = R.Dev(kv.reshape(c.tokens + 2, row), dt)
    K, V = (R.Dev(c.filled(t, LEFT), dt) for t in before)
    S, N, T = (R.Dev(t, abi.I32) for t in (c.starts, c.lens, c.table))
    f = frequencies(rotary) if rotary else None
    F = hb.DeviceBuffer.from_array(f) if rotary else None
    size = 4 if dt == abi.F32 else 2
    hb.paged_append(dt, KV.ptr, KV.ptr + 3 * 64 * size, S.ptr, N.ptr, T.ptr, K.ptr, V.ptr, 4, c.tokens + 2, 3, 64, row, c.pages,
                    page, c.width, F, rotary, interleaved, 1.5)
    hb.synchronize()
    kb = [np.zeros(t.shape) for t in before[0]]
    for s, (n, m) in enumerate(zip(lens, new)):
        x, at = kv[c.starts[s]:c.starts[s] + m], np.arange(n - m, n)
        k, e = A.rope(x[:, 0], at, f, rotary, interleaved, 1.5, dt) if rotary else (x[:, 0], np.zeros(x[:, 0].shape))
        before[0][s], kb[s] = np.concatenate([before[0][s], k]), np.concatenate([kb[s], e])
        before[1][s] = np.concatenate([before[1][s], x[:, 1]])
    wide = lambda rows, fill: _filled64(c, rows, fill)
    R.check(K.get(), wide(before[0], LEFT), wide(kb, 0.0), "keys")
    np.testing.assert_array_equal(V.get(), wide(before[1], LEFT))


def _filled64(c, rows, fill):
    out = np.full((c.pages, c.kv, c.page, c.d), fill)
    for s, r in enumerate(rows):
        for p in range(len(r)):
            out[c.table[s, p // c.page], :, p % c.page] = r[p]
    return out


def test_append_leaves_out_what_has_no_place():
    """Page numbers outside the pages, positions below 0 and past the table."""
    dt, kv = abi.BF16, R.rounded(synth.normal(5, (12, 1, 16)), abi.BF16)
    starts, lens = np.array([0, 4, 8, 12], np.int32), np.array([2, 34, 20], np.int32)
    table = np.array([[0, -9], [1, 2], [3, -1]], np.int32)
    K, V = (R.Dev(np.full((4, 1, 16, 16), LEFT), dt) for _ in range(2))
    X, S, N, T = R.Dev(kv, dt), *(R.Dev(t, abi.I32) for t in (starts, lens, table))
    hb.paged_append(dt, X.ptr, X.ptr, S.ptr, N.ptr, T.ptr, K.ptr, V.ptr, 3, 12, 1, 16, 16, 4, 16, 2)
    hb.synchronize()
    want = np.full((4, 1, 16, 16), LEFT)
    want[0, 0, 0], want[0, 0, 1] = kv[2, 0], kv[3, 0]     # positions -2, -1, 0, 1
    want[2, 0, 14], want[2, 0, 15] = kv[4, 0], kv[5, 0]   # positions 30 .. 33 of 32
    np.testing.assert_array_equal(K.get(), want)          # positions 16 .. 19 on page -1
    np.testing.assert_array_equal(V.get(), want)


@pytest.mark.parametrize("n,most", [(5000, 2), (5000, 4), (150, 3), (65, 40)])
def test_thousands_of_sequences(n, most):
    """More than 64 times 64, some without a new token: the append's places and the attention over them."""
    new = (synth.uniform01(8, n) * most).astype(int)
    lens = new + (synth.uniform01(9, n) * 20).astype(int)
    c = Cache(lens, new, 2, 1, 8, 16, abi.F32)
    got, (want, bound) = c.attend(0.3), c.want(0.3)
    R.check(got, want, bound, "o")
    rows = [t[len(t) - m:] for t, m in zip(c.k, new)]
    k = R.Dev(np.concatenate(rows + [np.full((2, 1, 8), LEFT, np.float32)]), abi.F32)
    K, V = (R.Dev(np.full((c.pages, 1, 16, 8), LEFT), abi.F32) for _ in range(2))
    S, N, T = (R.Dev(t, abi.I32) for t in (c.starts, c.lens, c.table))
    hb.paged_append(abi.F32, k.ptr, k.ptr, S.ptr, N.ptr, T.ptr, K.ptr, V.ptr, n, c.tokens + 2, 1, 8, 8, c.pages, 16, c.width)
    hb.synchronize()
    places = np.full((c.pages, 1, 16, 8), LEFT)
    for s, (r, m) in enumerate(zip(rows, new)):
        for j, p in enumerate(range(int(lens[s]) - int(m), int(lens[s]))):
            places[c.table[s, p // 16], :, p % 16] = r[j]
    np.testing.assert_array_equal(K.get(), places)
    np.testing.assert_array_equal(V.get(), places)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_steps_of_a_sequence_are_its_whole_attention(dt):
    """Prompts in one step, then chunks and single tokens through append and paged
    attention: every token's result is that of the whole sequence's attention."""
    from test_gpu_rope_rows import frequencies
    lens, heads, kv, dim, page = [75, 40], 4, 2, 32, 16
    x = [[R.rounded(synth.normal(9 + 3 * s + i, (n, h, dim)), dt) for i, h in enumerate((heads, kv, kv))]
         for s, n in enumerate(lens)]
    f = frequencies(dim)
    F = hb.DeviceBuffer.from_array(f)
    pages, width = 10, 5
    table = np.array([[7, 2, 9, 0, 4], [1, 8, 3, -1, -1]], np.int32)
    K, V = (R.Dev(np.full((pages, kv, page, dim), np.nan), dt) for _ in range(2))
    T = R.Dev(table, abi.I32)
    got = [np.zeros((n, heads, dim)) for n in lens]
    at = [0, 0]
    for step in ([50, 30], [20, 1], [1, 1], [4, 8]):
        starts = np.array([0, step[0], sum(step)], np.int32)
        now = np.array([a + n for a, n in zip(at, step)], np.int32)
        rows = [np.concatenate([x[s][i][at[s]:now[s]] for s in (0, 1)]) for i in range(3)]
        pos = np.concatenate([np.arange(at[s], now[s]) for s in (0, 1)]).astype(np.int32)
        n = sum(step)
        Q, NK, NV = (R.Dev(r, dt) for r in rows)
        S, N, P = (R.Dev(t, abi.I32) for t in (starts, now, pos))
        O = R.Dev(dt=dt, shape=(n, heads, dim))
        hb.rope_rows(dt, Q.ptr, P.ptr, F, Q.ptr, n, heads, dim, dim, heads * dim, heads * dim)
        hb.paged_append(dt, NK.ptr, NV.ptr, S.ptr, N.ptr, T.ptr, K.ptr, V.ptr, 2, n, kv, dim, kv * dim, pages, page, width, F, dim)
        hb.paged_attention(dt, Q.ptr, K.ptr, V.ptr, S.ptr, N.ptr, T.ptr, O.ptr, 2, n, heads, kv, dim, heads * dim, heads * dim,
                           pages, page, width, dim ** -0.5)
        hb.synchronize()
        o = O.get()
        for s in (0, 1):
            got[s][at[s]:now[s]] = o[starts[s]:starts[s + 1]]
        at = list(now)
    for s, n in enumerate(lens):
        pos = np.arange(n)
        # The stored type's rounding of the turned rows, then the attention of those.
        turned = [A.rope(t, pos, f, dim, False, 1.0, dt)[0] for t in x[s][:2]]
        q, k = (R.rounded(t.astype(np.float32), dt).astype(np.float64) for t in turned)
        for h in range(heads):
            o, e, *_ = A.attend(q[:, h], k[:, h // 2], x[s][2][:, h // 2].astype(np.float64), 0, dim ** -0.5, True, dt)
            # A value turned in f32 may round to the other neighbour: one step of q and k, 2 HALF of either.
            z = np.abs(q[:, h]) @ np.abs(k[:, h // 2]).T * dim ** -0.5
            e = e + 8 * R.HALF[dt] * z.max(1, keepdims=True) * np.abs(x[s][2][:, h // 2]).max()
            R.check(got[s][:, h], o, e, f"sequence {s} head {h}")


@pytest.mark.parametrize("new", [1, 60])
def test_same_bits_on_another_stream_and_replayed(new):
    c = Cache([900, 1400], [new, 1], 8, 2, 64, 16, abi.BF16)
    one = c.attend(0.2)
    s = hb.create_stream()
    try:
        np.testing.assert_array_equal(one, c.attend(0.2, stream=s))
        K, V, Q = (R.Dev(t, c.dt) for t in (c.filled(c.k), c.filled(c.v), c.q))
        S, N, T = (R.Dev(t, abi.I32) for t in (c.starts, c.lens, c.table))
        O = R.Dev(dt=c.dt, shape=c.q.shape)
        args = (c.dt, Q.ptr, K.ptr, V.ptr, S.ptr, N.ptr, T.ptr, O.ptr, 2, c.tokens, 8, 2, 64, 512, 512, c.pages, 16, c.width, 0.2)
        with hb.Graph(s) as g:
            hb.paged_attention(*args, s)
        for _ in range(3):
            g.launch()
            np.testing.assert_array_equal(one, c.attend(0.2))  # eager work of the null stream
            hb.synchronize(s)
            np.testing.assert_array_equal(one, O.get())
        # The lengths live on the device: a replay takes new ones.
        shorter = np.array([700, 1300], np.int32)
        N.buf.upload(shorter, N.at)
        c.lens = shorter
        c.k, c.v = ([t[:n] for t, n in zip(x, shorter)] for x in (c.k, c.v))
        g.launch()
        hb.synchronize(s)
        R.check(O.get(), *c.want(0.2), "shorter")
        g.close()
    finally:
        hb.destroy_stream(s)


def test_pages_beyond_32_bits():
    """Pages of 1 MiB, 4.6 GB of them: a sequence on the last ones, its rows appended there too."""
    dt, page, pages, n = abi.F16, 4096, 4600, 5000
    k, v = (R.rounded(synth.normal(i, (n, 1, 128)), dt) for i in (1, 2))
    q = R.rounded(synth.normal(3, (2, 4, 128)), dt)
    K, V = (hb.DeviceBuffer(pages * page * 128 * 2) for _ in range(2))
    table = np.array([[4599, 4501]], np.int32)
    T, S, N = R.Dev(table, abi.I32), R.Dev(np.array([0, 2], np.int32), abi.I32), R.Dev(np.array([n], np.int32), abi.I32)
    for dev, rows in ((K, k), (V, v)):
        for i, p in enumerate(table[0]):
            dev.upload(synth.f16_bits(rows[page * i:min(page * (i + 1), n - 2)].reshape(-1)), int(p) * page * 128 * 2)
    X, Y, Q, O = R.Dev(k[-2:], dt), R.Dev(v[-2:], dt), R.Dev(q, dt), R.Dev(dt=dt, shape=q.shape)
    hb.paged_append(dt, X.ptr, Y.ptr, S.ptr, N.ptr, T.ptr, K, V, 1, 2, 1, 128, 128, pages, page, 2)
    hb.paged_attention(dt, Q.ptr, K, V, S.ptr, N.ptr, T.ptr, O.ptr, 1, 2, 4, 1, 128, 512, 512, pages, page, 2, 0.1)
    hb.synchronize()
    got = O.get()
    for h in range(4):
        o, e, *_ = A.attend(*(t.astype(np.float64) for t in (q[:, h], k[:, 0], v[:, 0])), n - 2, 0.1, True, dt)
        R.check(got[:, h], o, e, f"head {h}")
    K.free()
    V.free()
