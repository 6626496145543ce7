"""Scaled embedding rows and their gradient against 64 bits, within the bounds
of operators_ref.py."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


def words(seed, n, vocab):
    """Ids as frequent as words: P(id) about 1 / (id + 1)."""
    u = synth.uniform01(seed, n)
    return np.minimum(np.exp(u * np.log(vocab + 1.0)) - 1, vocab - 1).astype(np.int32)


def forward(w, ids, scale, dt, offset=0):
    W, I = R.Dev(w, dt, offset), R.Dev(ids, abi.I32)
    Y = R.Dev(dt=dt, offset=offset, shape=(len(ids), w.shape[1]))
    hb.embedding_rows(dt, W.ptr, I.ptr, Y.ptr, len(ids), *w.shape, scale)
    hb.synchronize()
    return Y.get()


def gradient(dy, ids, vocab, scale, dt, offset=0, stream=None):
    G, I = R.Dev(dy, dt, offset), R.Dev(ids, abi.I32)
    D = R.Dev(dt=dt, offset=offset, shape=(vocab, dy.shape[1]))
    hb.embedding_vjp_rows(dt, G.ptr, I.ptr, D.ptr, len(ids), vocab, dy.shape[1], scale, stream)
    hb.synchronize(stream)
    return D.get()


SIZES = [(1, 1, 1), (1, 5, 7), (3, 2, 8), (8, 32000, 768), (64, 10, 64), (65, 300, 65), (1000, 1, 33), (1023, 257, 40),
         (1025, 70000, 24), (1537, 3203, 777), (2048, 256, 1024), (5000, 50257, 16), (16384, 1000, 8),
         (16385, 1000, 8), (40000, 300, 20), (50001, 70000, 8)]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("n,vocab,dim", SIZES)
def test_matches_64_bits(n, vocab, dim, dt):
    print(f"embedding {n} of {vocab}x{dim} {R.NAMES[dt]}", flush=True)
    ids, scale = words(n + vocab, n, vocab), dim ** 0.5
    if n < 10000:
        w = R.rounded(synth.normal(vocab, (vocab, dim)), dt)
        R.check(forward(w, ids, scale, dt), *R.embedding(w, ids, scale, dt), f"y {n} {vocab} {dim}")
    dy = R.rounded(synth.normal(n, (n, dim)), dt)
    R.check(gradient(dy, ids, vocab, scale, dt), *R.embedding_vjp(dy, ids, vocab, scale, dt), f"dw {n} {vocab} {dim}")


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("dim,offset", [(777, 1), (64, 3), (7, 5)])
@pytest.mark.parametrize("n", [50, 300])
def test_any_element_alignment(n, dim, offset, dt):
    ids = words(5, n, 50)
    w, dy = R.rounded(synth.normal(1, (50, dim)), dt), R.rounded(synth.normal(2, (n, dim)), dt)
    R.check(forward(w, ids, 0.25, dt, offset), *R.embedding(w, ids, 0.25, dt), "y")
    R.check(gradient(dy, ids, 50, 0.25, dt, offset), *R.embedding_vjp(dy, ids, 50, 0.25, dt), "dw")


@pytest.mark.parametrize("n", [5, 60, 4000, 20000])
def test_ids_out_of_range_are_clamped(n):
    ids = words(9, n, 40)
    ids[::5] = -1
    ids[1::7] = 40
    ids[2::11] = np.iinfo(np.int32).max
    ids[3::13] = np.iinfo(np.int32).min
    w, dy = synth.normal(1, (40, 24)), synth.normal(2, (n, 24))
    R.check(forward(w, ids, 2.0, abi.F32), *R.embedding(w, ids, 2.0, abi.F32), "y")
    R.check(gradient(dy, ids, 40, 2.0, abi.F32), *R.embedding_vjp(dy, ids, 40, 2.0, abi.F32), "dw")


@pytest.mark.parametrize("n", [1, 3, 63, 64, 65, 2000, 16384, 30000])
@pytest.mark.parametrize("kind", ["one id", "descending", "each once", "two ids"])
def test_runs_across_every_share(n, kind):
    """All positions one id (a run across every share), every id once, orders
    that the sort has to turn round."""
    vocab = 30011
    ids = {"one id": np.full(n, 17), "descending": vocab - 1 - np.arange(n) % vocab, "each once": np.arange(n) % vocab,
           "two ids": np.arange(n) % 2 * 300}[kind].astype(np.int32)
    dy = synth.normal(n, (n, 12))
    R.check(gradient(dy, ids, vocab, 1.0, abi.F32), *R.embedding_vjp(dy, ids, vocab, 1.0, abi.F32), kind)


@pytest.mark.parametrize("n", [3000, 20000])
def test_equal_ids_are_summed_in_the_order_of_their_positions(n):
    """A 1 and then 2^-24 (half its last place) everywhere: in the order of the
    positions the first share adds nothing to its 1, any other order does. The
    shares' sums (exact but the first) are then joined in order too, in four
    contiguous parts where there are more than 16 of them behind the first."""
    ids = np.zeros(n, np.int32)
    dy = np.full((n, 8), 2.0 ** -24, np.float32)
    dy[0] = 1.0
    got = gradient(dy, ids, 3, 1.0, abi.F32)
    share = max(-(-n // 2048), 4)
    sums = [np.float32((min(n, lo + share) - lo) * 2.0 ** -24) for lo in range(0, n, share)]
    sums[0] = np.float32(1.0)
    each = -(-(len(sums) - 1) // 4)
    parts = []
    for w in range(4):
        acc = sums[0] if w == 0 else np.float32(0)
        for v in sums[1 + w * each:1 + (w + 1) * each]:
            acc = np.float32(acc + v)
        parts.append(acc)
    acc = parts[0]
    for v in parts[1:]:
        acc = np.float32(acc + v)
    np.testing.assert_array_equal(got[0], np.full(8, acc, np.float64))
    assert not got[1:].any()


def test_non_finite_rows_stay_with_their_ids():
    ids = words(3, 500, 30)
    dy = synth.normal(4, (500, 16))
    dy[np.flatnonzero(ids == 2)[0]] = np.nan
    dy[np.flatnonzero(ids == 5)[0]] = np.inf
    got = gradient(dy, ids, 30, 1.0, abi.F32)
    assert np.isnan(got[2]).all() and np.isposinf(got[5]).all()
    rest = [i for i in range(30) if i not in (2, 5)]
    want, bound = R.embedding_vjp(np.where(np.isfinite(dy), dy, 0), ids, 30, 1.0, abi.F32)
    R.check(got[rest], want[rest], bound[rest], "other rows")


def test_no_tokens():
    D = R.Dev(dt=abi.F16, shape=(31, 7), offset=1)
    hb.embedding_vjp_rows(abi.F16, 0, 0, D.ptr, 0, 31, 7, 1.0)
    hb.embedding_rows(abi.F16, 0, 0, 0, 0, 31, 7, 1.0)
    hb.synchronize()
    assert not D.get().any()


@pytest.mark.parametrize("n", [60, 900, 25000])
def test_same_bits_every_time_and_on_another_stream(n):
    ids, dy = words(3, n, 5000), R.rounded(synth.normal(4, (n, 100)), abi.BF16)
    one = gradient(dy, ids, 5000, 3.0, abi.BF16)
    s = hb.create_stream()
    try:
        for stream in (None, s):
            np.testing.assert_array_equal(one, gradient(dy, ids, 5000, 3.0, abi.BF16, stream=stream))
    finally:
        hb.destroy_stream(s)
