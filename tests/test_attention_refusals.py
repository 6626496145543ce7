"""Arguments that the rotary, packed and paged attention entry points refuse: every
check runs before any device call, so these hold without a GPU."""
import pytest

from oxidizedmlx_amd import abi
from oxidizedmlx_amd import backend as hb

P = 4096  # an aligned address that no call reaches
BIG = 1 << 31
NAN, INF = float("nan"), float("inf")


def freqs(freqs=P, rotary=8, base=10000.0, factor=1.0, low=0.0, high=0.0, original=0):
    hb.rope_frequencies(freqs, rotary, base, factor, low, high, original)


def rope(f=hb.rope_rows, dt=abi.F32, x=P, pos=P, freqs=P, y=P, tokens=2, heads=2, dim=8, rotary=8, xs=16, ys=16, inter=0):
    f(dt, x, pos, freqs, y, tokens, heads, dim, rotary, xs, ys, inter)


def rope_vjp(**kw):
    rope(hb.rope_vjp_rows, **kw)


def packed(dt=abi.F32, q=P, k=P, v=P, starts=P, o=P, lse=P, seqs=1, tokens=4, heads=4, kv=2, dim=8, qs=32, ks=16, os=32,
           scale=1.0):
    hb.packed_attention(dt, q, k, v, starts, o, lse, seqs, tokens, heads, kv, dim, qs, ks, os, scale)


def packed_vjp(dt=abi.F32, q=P, k=P, v=P, o=P, g=P, lse=P, starts=P, dq=P, dk=P, dv=P, seqs=1, tokens=4, heads=4, kv=2, dim=8,
               qs=32, ks=16, os=32, scale=1.0):
    hb.packed_attention_vjp(dt, q, k, v, o, g, lse, starts, dq, dk, dv, seqs, tokens, heads, kv, dim, qs, ks, os, scale)


def append(dt=abi.F32, k=P, v=P, starts=P, lens=P, table=P, kp=P, vp=P, seqs=1, tokens=4, kv=2, dim=8, ks=16, pages=3, page=16,
           width=2, freqs=None, rotary=0, inter=0):
    hb.paged_append(dt, k, v, starts, lens, table, kp, vp, seqs, tokens, kv, dim, ks, pages, page, width, freqs, rotary, inter)


def paged(dt=abi.F32, q=P, kp=P, vp=P, starts=P, lens=P, table=P, o=P, seqs=1, tokens=4, heads=4, kv=2, dim=8, qs=32, os=32,
          pages=3, page=16, width=2, scale=1.0):
    hb.paged_attention(dt, q, kp, vp, starts, lens, table, o, seqs, tokens, heads, kv, dim, qs, os, pages, page, width, scale)


ALL = [freqs, rope, rope_vjp, packed, packed_vjp, append, paged]
POINTERS = [(freqs, "freqs"), (rope, "x pos freqs y"), (rope_vjp, "x pos freqs y"), (packed, "q k v starts o"),
            (packed_vjp, "q k v o g lse starts dq dk dv"), (append, "k v starts lens table kp vp"),
            (paged, "q kp vp starts lens table o")]
CASES = [(f, k) for f, names in POINTERS for k in names.split()]
ids = lambda v: v if isinstance(v, str) else getattr(v, "__name__", "")


@pytest.mark.parametrize("f,name", CASES, ids=ids)
def test_null_operands(f, name):
    with pytest.raises(abi.NullPtr):
        f(**{name: 0})


@pytest.mark.parametrize("f,name", CASES + [(packed, "lse")], ids=ids)
def test_unaligned_operands(f, name):
    for off in ((1, 2, 3) if f in (rope, rope_vjp) or name in ("starts", "lens", "table", "lse") else (2, 4) if name == "freqs" else (4, 8)):
        with pytest.raises(abi.InvalidArgument, match="aligned"):
            f(**{name: P + off})
    if name in ("x", "y"):
        with pytest.raises(abi.InvalidArgument, match="aligned"):
            f(dt=abi.BF16, **{name: P + 1})


def test_unaligned_frequencies_of_an_append():
    with pytest.raises(abi.InvalidArgument, match="aligned"):
        append(freqs=P + 4, rotary=8)


@pytest.mark.parametrize("f", ALL[1:], ids=ids)
@pytest.mark.parametrize("dt", [abi.I32, abi.I64, -1, 99])
def test_other_types(f, dt):
    with pytest.raises(abi.InvalidArgument, match="dtype"):
        f(dt=dt)


HEADS = [{"dim": 12}, {"dim": 136}, {"dim": -8}, {"kv": 0}, {"kv": -1}, {"seqs": -1}, {"tokens": -1}, {"seqs": (1 << 20) + 1},
         {"tokens": (1 << 29) + 1}]
SIZES = [
    (freqs, [{"rotary": 0}, {"rotary": 7}, {"rotary": 1026}, {"rotary": -2}, {"base": 0.0}, {"base": NAN}, {"base": INF},
             {"factor": 0.0}, {"factor": -1.0}, {"factor": NAN}, {"original": -1}, {"factor": 2.0, "original": 4096},
             {"factor": 2.0, "original": 4096, "low": 4.0, "high": 1.0}, {"factor": 2.0, "original": 4096, "low": NAN, "high": 1.0}]),
    (packed, HEADS + [{"heads": 5}, {"heads": -4}, {"qs": 28}, {"ks": 12}, {"os": 28}, {"qs": 33}, {"ks": 18}, {"os": 34},
                      {"qs": (1 << 20) + 4}, {"dt": abi.BF16, "qs": 36}, {"scale": NAN}, {"scale": INF},
                      {"tokens": (1 << 27) + 1}]),
    (append, HEADS[:3] + HEADS[4:] + [{"ks": 12}, {"ks": 18}, {"tokens": (1 << 24) + 1}, {"page": 8}, {"page": 24}, {"page": 0},
                          {"page": 8192}, {"page": -16}, {"pages": -1}, {"pages": BIG}, {"width": -1},
                          {"width": (1 << 26) + 1}, {"freqs": P, "rotary": 9}, {"freqs": P, "rotary": 16}, {"freqs": P, "rotary": 0},
                          {"freqs": P, "rotary": 8, "inter": 2}]),
    (paged, HEADS + [{"heads": 5}, {"qs": 28}, {"os": 28}, {"qs": 33}, {"page": 8}, {"page": 48}, {"page": 8192},
                     {"pages": 0}, {"pages": -1}, {"width": 0}, {"width": -1}, {"width": (1 << 26) + 1}, {"scale": NAN},
                     {"tokens": (1 << 27) + 1}]),
]
SIZES.append((packed_vjp, SIZES[1][1]))
for f in (rope, rope_vjp):
    SIZES.append((f, [{"tokens": -1}, {"heads": -1}, {"dim": -1}, {"rotary": 10}, {"rotary": 7}, {"rotary": 0}, {"xs": 15},
                      {"ys": 15}, {"xs": (1 << 20) + 1}, {"tokens": (1 << 24) + 1}, {"heads": 1 << 18, "xs": 1 << 20, "ys": 1 << 20},
                      {"inter": 2}, {"inter": -1}, {"xs": 17}, {"ys": 17}]))


@pytest.mark.parametrize("f,sizes", SIZES, ids=ids)
def test_sizes(f, sizes):
    for kw in sizes:
        with pytest.raises(abi.InvalidArgument):
            f(**kw)
            pytest.fail(f"{f.__name__} takes {kw}")


def test_nothing_to_do_needs_no_device():
    rope(tokens=0, x=0, pos=0, freqs=0, y=0)
    rope_vjp(heads=0, x=0, pos=0, freqs=0, y=0)
    packed(tokens=0, q=0, k=0, v=0, starts=0, o=0)
    packed(seqs=0, q=0, k=0, v=0, starts=0, o=0)
    packed(heads=0, kv=0, q=0)
    packed_vjp(tokens=0, q=0, dq=0)
    append(tokens=0, k=0)
    append(pages=0, kp=0, vp=0)
    append(width=0, table=0)
    paged(tokens=0, q=0)
    paged(seqs=0, q=0, starts=0)


@pytest.mark.parametrize("f", ALL, ids=ids)
def test_a_sound_call_wants_the_device(f):
    if hb.device_count() > 0:
        pytest.skip("a GPU is present")
    with pytest.raises(abi.BackendUnavailable):
        f()
