"""Arguments that the affine layer norm, embedding and linear cross entropy
entry points refuse: every check runs before any device call, so these hold
without a GPU."""
import pytest

from oxidizedmlx_amd import abi
from oxidizedmlx_amd import backend as hb

P = 4096  # an aligned address that no call reaches
BIG = 1 << 31
ROW = (1 << 23) + 1


def ln(dt=abi.F32, x=P, w=P, b=P, y=P, rows=2, cols=8):
    hb.layernorm_affine_rows(dt, x, w, b, y, rows, cols, 1e-5)


def ln_vjp(dt=abi.F32, dy=P, x=P, w=P, dx=P, dw=P, db=P, rows=2, cols=8):
    hb.layernorm_affine_vjp_rows(dt, dy, x, w, dx, dw, db, rows, cols, 1e-5)


def emb(dt=abi.F32, w=P, ids=P, y=P, n=2, vocab=5, dim=8):
    hb.embedding_rows(dt, w, ids, y, n, vocab, dim, 1.0)


def emb_vjp(dt=abi.F32, dy=P, ids=P, dw=P, n=2, vocab=5, dim=8):
    hb.embedding_vjp_rows(dt, dy, ids, dw, n, vocab, dim, 1.0)


def ce(dt=abi.F32, x=P, w=P, t=P, loss=P, lse=P, rows=2, dim=8, vocab=5):
    hb.linear_cross_entropy(dt, x, w, t, loss, lse, rows, dim, vocab)


def ce_vjp(dt=abi.F32, x=P, w=P, t=P, lse=P, g=P, dx=P, dw=P, rows=2, dim=8, vocab=5):
    hb.linear_cross_entropy_vjp(dt, x, w, t, lse, g, dx, dw, rows, dim, vocab)


POINTERS = [(ln, "x w b y"), (ln_vjp, "dy x w dx dw db"), (emb, "w ids y"), (emb_vjp, "dy ids dw"),
            (ce, "x w t loss lse"), (ce_vjp, "x w t lse g")]
CASES = [(f, k) for f, names in POINTERS for k in names.split()]


@pytest.mark.parametrize("f,name", CASES, ids=lambda v: v if isinstance(v, str) else v.__name__)
def test_null_operands(f, name):
    with pytest.raises(abi.NullPtr):
        f(**{name: 0})


@pytest.mark.parametrize("f,name", CASES + [(ce_vjp, "dx"), (ce_vjp, "dw")],
                         ids=lambda v: v if isinstance(v, str) else v.__name__)
def test_unaligned_operands(f, name):
    with pytest.raises(abi.InvalidArgument, match="aligned"):
        f(**{name: P + 2})
    if name not in ("ids", "t", "loss", "lse", "g"):
        with pytest.raises(abi.InvalidArgument, match="aligned"):
            f(dt=abi.BF16, **{name: P + 1})


@pytest.mark.parametrize("f", [ln, ln_vjp, emb, emb_vjp, ce, ce_vjp], ids=lambda f: f.__name__)
@pytest.mark.parametrize("dt", [abi.I32, abi.I64, -1, 99])
def test_other_types(f, dt):
    with pytest.raises(abi.InvalidArgument, match="dtype"):
        f(dt=dt)


@pytest.mark.parametrize("f,sizes", [
    (ln, [{"rows": -1}, {"cols": -1}, {"rows": BIG}, {"cols": ROW}]),
    (ln_vjp, [{"rows": -1}, {"cols": -1}, {"rows": BIG}, {"cols": ROW}]),
    (emb, [{"n": -1}, {"vocab": -1}, {"dim": -1}, {"n": BIG}, {"vocab": BIG}, {"dim": (1 << 20) + 1},
           {"vocab": 0}]),
    (emb_vjp, [{"n": -1}, {"vocab": -1}, {"dim": -1}, {"n": BIG}, {"vocab": BIG}, {"dim": (1 << 20) + 1},
               {"vocab": 0}]),
    (ce, [{"rows": -1}, {"dim": -1}, {"vocab": -1}, {"rows": BIG}, {"vocab": BIG}, {"dim": (1 << 20) + 1}, {"dim": 0},
          {"vocab": 0}, {"rows": 1 << 12, "dim": 1 << 19}]),
    (ce_vjp, [{"rows": -1}, {"dim": -1}, {"vocab": -1}, {"rows": BIG}, {"vocab": BIG}, {"dim": (1 << 20) + 1}, {"dim": 0},
              {"vocab": 0}, {"rows": 1 << 12, "dim": 1 << 19}]),
], ids=lambda v: v.__name__ if callable(v) else "")
def test_sizes(f, sizes):
    for kw in sizes:
        with pytest.raises(abi.InvalidArgument):
            f(**kw)


def test_nothing_to_do_needs_no_device():
    ln(rows=0, x=0, y=0, w=0, b=0)
    ln(cols=0)
    ln_vjp(cols=0)
    emb(n=0, w=0, ids=0, y=0)
    emb(dim=0)
    emb_vjp(dim=0)
    emb_vjp(n=0, vocab=0)
    ce(rows=0, x=0, w=0, t=0, loss=0, lse=0)
    ce_vjp(dx=0, dw=0)


@pytest.mark.parametrize("f", [ln, ln_vjp, emb, emb_vjp, ce, ce_vjp], ids=lambda f: f.__name__)
def test_a_sound_call_wants_the_device(f):
    if hb.device_count() > 0:
        pytest.skip("a GPU is present")
    with pytest.raises(abi.BackendUnavailable):
        f()
