"""Linear cross entropy over several pieces of the vocabulary, and the loops of its
few-row kernels that long rows take, each counted or sized so that they run."""
import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi
from oxidizedmlx_amd import backend as hb
from test_gpu_cross_entropy import inputs
from test_gpu_cross_entropy_range import check_all, forward, run

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


@pytest.fixture
def pieces():
    """Sets the bytes of a piece and returns how many pieces ran since."""
    set_bytes = hb.lib().mlxhip_debug_cross_entropy_pieces
    set_bytes(0)
    yield set_bytes
    set_bytes(0)


def spread_targets(t, vocab):
    """Counted targets in the first, the middle and the last columns among them."""
    on = np.flatnonzero((t >= 0) & (t < vocab))
    t[on[:4]] = 0, vocab // 2, vocab - 1, 256
    return t


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rows,dim,vocab,least", [(70, 72, 700, 3), (130, 77, 1300, 6), (300, 264, 1025, 5), (65, 40, 257, 2),
                                                  (600, 96, 777, 4)])
def test_pieces_of_256_columns(pieces, rows, dim, vocab, least, offset, dt):
    """Copied (ragged or offset) and in-place W, a last piece shorter than the
    others, targets in each."""
    x, w, t, g = inputs(rows, dim, vocab, dt)
    t = spread_targets(t, vocab)
    pieces(1)
    got = run(x, w, t, g, dt, offset)
    ran = pieces(1)
    forward_splits = dt == abi.F32 and rows > 128 or dt != abi.F32 and (dim % 8 or offset) and rows > 64
    assert ran >= least + (least if forward_splits else 0), ran
    check_all(got, x, w, t, g, dt)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_a_piece_of_several_tiles(pieces, dt):
    """Pieces of 768 of 2000 columns: dx's slices of K in each, fewer in the last."""
    rows, dim, vocab = 140, 264, 2000
    x, w, t, g = inputs(rows, dim, vocab, dt)
    t = spread_targets(t, vocab)
    pieces(rows * 900 * 2 * (3 if dt == abi.F32 else 2))
    got = run(x, w, t, g, dt)
    assert pieces(0) >= 3
    check_all(got, x, w, t, g, dt)


@pytest.mark.parametrize("dt", [abi.BF16, abi.F16], ids=R.NAMES.get)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rows,dim,vocab", [(17, 131, 600), (40, 77, 700), (64, 390, 515)])
def test_pieces_of_rows_whose_logits_come_straight_from_w(pieces, rows, dim, vocab, offset, dt):
    x, w, t, g = inputs(rows, dim, vocab, dt)
    t = spread_targets(t, vocab)
    pieces(1)
    got = run(x, w, t, g, dt, offset)
    assert pieces(0) >= 3
    check_all(got, x, w, t, g, dt)


@pytest.mark.parametrize("rows,dim,dt", [(200, 72, dt) for dt in R.DTYPES] + [(100, 77, dt) for dt in R.DTYPES] +
                         [(24, 77, abi.BF16), (24, 77, abi.F16)])
@pytest.mark.parametrize("want", ["x", "w"])
def test_one_gradient_alone_in_pieces(pieces, want, rows, dim, dt):
    a = inputs(rows, dim, 700, dt)
    pieces(1)
    both = run(*a, dt)
    pieces(1)
    one = run(*a, dt, want=want)
    assert pieces(0) >= 3
    i = 2 if want == "x" else 3
    np.testing.assert_array_equal(one[i], both[i])


def test_the_default_pieces_split_a_large_w(pieces):
    """W's planes of 130 f32 rows' loss over 140000 x 1024 take 573 MB: two pieces."""
    x, w, t, _ = inputs(130, 1024, 140000, abi.F32)
    t = spread_targets(t, 140000)
    X, W, T = R.Dev(x), R.Dev(w), R.Dev(t, abi.I32)
    L, S = R.Dev(shape=(130,)), R.Dev(shape=(130,))
    hb.linear_cross_entropy(abi.F32, X.ptr, W.ptr, T.ptr, L.ptr, S.ptr, 130, 1024, 140000)
    hb.synchronize()
    assert pieces(0) == 2
    for name, a, (v, b) in zip(("loss", "lse"), (L.get(), S.get()), forward(x, w, t, abi.F32)):
        R.check(a, v, b, name)


# 16-bit losses of 17 to 64 rows read W as it is where its rows are no whole 16-byte
# chunks or begin off one: batches of 128 (to 32 rows) or 96 columns in two buffers in
# turn, whole blocks of 32 behind them and a last one that is not whole.
LONG = [(20, 131), (32, 390), (17, 520), (24, 260), (31, 134), (40, 101), (64, 295), (50, 198), (33, 484), (64, 676)]


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("rows,dim", LONG)
def test_few_rows_of_many_columns(rows, dim, offset, dt):
    a = inputs(rows, dim, 515, dt)
    check_all(run(*a, dt, offset), *a, dt)


@pytest.mark.parametrize("dt", [abi.BF16, abi.F16], ids=R.NAMES.get)
@pytest.mark.parametrize("rows", [1, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("dim", [96, 128, 192, 256, 384, 1152])
def test_few_rows_of_aligned_columns_off_their_chunks(rows, dim, dt):
    """Whole batches without a tail, every row off a 16-byte chunk by one element."""
    a = inputs(rows, dim, 300, dt)
    check_all(run(*a, dt, 1), *a, dt)
