"""Plain 64-bit forms of the embedding, affine layer norm and linear cross
entropy operators, the error bounds of their f32 / 16-bit kernels, and device
arrays with guard elements around them.

Bounds: u = 2^-24 is half an f32 step, ``half(dt)`` half a step of the stored
type. A sum of n f32 terms is off by at most (its depth) * u * sum of their
magnitudes; depths are given where they are used."""
import numpy as np

from oxidizedmlx_amd import abi
from oxidizedmlx_amd import backend as hb
from oxidizedmlx_amd import synth

U = 2.0 ** -24
HALF = {abi.F32: 2.0 ** -24, abi.BF16: 2.0 ** -8, abi.F16: 2.0 ** -11}
# What is lost near zero: half the f16 subnormals' step; f32 and bf16 values
# below the smallest normal one, 2^-126, may become 0.
NORMAL = 2.0 ** -126
TINY = {abi.F32: NORMAL, abi.BF16: NORMAL, abi.F16: 2.0 ** -25}
NAMES = {abi.F32: "f32", abi.BF16: "bf16", abi.F16: "f16"}
DTYPES = [abi.F32, abi.BF16, abi.F16]
GUARD = 0x5A


def rounded(a, dt):
    """The values of f32 array ``a`` as the type holds them (as float32)."""
    return a if dt == abi.F32 else synth.round_bf16(a) if dt == abi.BF16 else synth.round_f16(a)


class Dev:
    """A device array of the type's elements, ``offset`` elements past a
    256-byte boundary, 64 guard bytes and more behind it."""

    def __init__(self, values=None, dt=abi.F32, offset=0, shape=None):
        self.shape = tuple(np.shape(values)) if values is not None else tuple(shape)
        self.dt, self.size = dt, 2 if dt in (abi.BF16, abi.F16) else 4
        self.n = int(np.prod(self.shape))
        self.at = offset * self.size
        host = np.full(self.at + self.n * self.size + 64, GUARD, np.uint8)
        if values is not None:
            host[self.at:self.at + self.n * self.size] = self._bits(values).view(np.uint8).reshape(-1)
        self.buf = hb.DeviceBuffer.from_array(host)
        self.ptr = self.buf.ptr + self.at

    def _bits(self, values):
        if self.dt == abi.I32:
            return np.ascontiguousarray(values, np.int32).reshape(-1)
        v = np.ascontiguousarray(values, np.float32).reshape(-1)
        return v if self.dt == abi.F32 else synth.bf16_bits(v) if self.dt == abi.BF16 else synth.f16_bits(v)

    def get(self):
        """The values as float64; the guards must be as they were."""
        raw = self.buf.download(np.uint8)
        assert (raw[:self.at] == GUARD).all() and (raw[self.at + self.n * self.size:] == GUARD).all(), "guard written"
        b = raw[self.at:self.at + self.n * self.size].copy()
        if self.dt == abi.F32:
            v = b.view(np.float32)
        elif self.dt == abi.BF16:
            v = synth.bf16_to_f32(b.view(np.uint16))
        else:
            v = b.view(np.float16)
        return v.astype(np.float64).reshape(self.shape)


def check(got, want, bound, what):
    """|got - want| <= bound everywhere; equal where the value is no finite number."""
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    np.testing.assert_array_equal(got[~fine], want[~fine], err_msg=what)
    off = np.abs(got - want)[fine]
    over = off > np.broadcast_to(bound, want.shape)[fine]
    worst = float((off / np.maximum(np.broadcast_to(bound, want.shape)[fine], 1e-300)).max()) if off.size else 0.0
    print(f"{what}: worst {worst:.3f} of the bound", flush=True)
    assert not over.any(), f"{what}: {int(over.sum())} of {off.size} values over the bound, by up to {worst:.2f} times"


# ── layer norm with weight and bias ───────────────────────────────────────

# Depth of a row's sum: at most 16 values of a lane in registers (rows of up to
# 16384; a longer row's lane adds cols / 1024), 6 steps of a wave, 16 waves.
def _row_depth(cols):
    return max(16, cols // 1024 + 1) + 6 + 16


def layer_norm(x, w, b, eps, dt):
    """y and its bound."""
    x, w, b = (np.asarray(a, np.float64) for a in (x, w, b))
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    xh = (x - mean) * rstd
    y = xh * w + b
    e = xh_error(x, xh, rstd)
    return y, (np.abs(w) * e + 2 * U * (np.abs(xh * w) + np.abs(y))) * (1 + HALF[dt]) + HALF[dt] * np.abs(y) + TINY[dt]


def xh_error(x, xh, rstd):
    """The mean is off by depth * u of the mean magnitude, which moves every
    deviation; rstd by half of the variance's relative error (depth + 2 * u for
    squares of rounded deviations) and three roundings; xh by its own two."""
    d = _row_depth(x.shape[1])
    return rstd * d * U * np.abs(x).mean(1, keepdims=True) + (d / 2 + 8) * U * np.abs(xh)


def layer_norm_vjp(dy, x, w, eps, dt):
    """(dx, dw, db) and their bounds."""
    dy, x, w = (np.asarray(a, np.float64) for a in (dy, x, w))
    rows, cols = x.shape
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    xh = (x - mean) * rstd
    g = dy * w
    c1, c2 = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    dx = rstd * (g - c1 - xh * c2)
    e, d = xh_error(x, xh, rstd), _row_depth(cols)
    m = np.abs(g).mean(1, keepdims=True)
    e2 = (d + 6) * U * np.abs(g * xh).mean(1, keepdims=True) + (np.abs(g) * e).mean(1, keepdims=True)
    terms = np.abs(g) + np.abs(c1) + np.abs(xh * c2)
    edx = rstd * (4 * U * terms + (d + 2) * U * m + np.abs(xh) * e2 + e * np.abs(c2)) + (d / 2 + 8) * U * rstd * terms
    # A column's sum: the rows of a workgroup (of 256, 64 for rows over 16384)
    # in order, four waves, an eighth of the workgroups, eight of those.
    groups = 256 if cols <= 16384 else 64
    n = rows // groups + 1 + 4 + groups // 8 + 8
    dw, db = (dy * xh).sum(0), dy.sum(0)
    edw = (n + 2) * U * np.abs(dy * xh).sum(0) + (np.abs(dy) * e).sum(0)
    edb = n * U * np.abs(dy).sum(0)
    return [(v, b * (1 + HALF[dt]) + HALF[dt] * np.abs(v) + TINY[dt]) for v, b in ((dx, edx), (dw, edw), (db, edb))]


# ── embedding ─────────────────────────────────────────────────────────────

def embedding(w, ids, scale, dt):
    y = np.asarray(w, np.float64)[np.clip(ids, 0, len(w) - 1)] * float(np.float32(scale))
    return y, (HALF[dt] + 2 * U) * np.abs(y) + TINY[dt]


def embedding_vjp(dy, ids, vocab, scale, dt):
    """A sum of `count` rows in order (in shares: no deeper), one product."""
    dy, at = np.asarray(dy, np.float64), np.clip(ids, 0, vocab - 1)
    dw, mag = np.zeros((vocab, dy.shape[1])), np.zeros((vocab, dy.shape[1]))
    np.add.at(dw, at, dy)
    np.add.at(mag, at, np.abs(dy))
    count = np.bincount(at, minlength=vocab)[:, None]
    s = float(np.float32(scale))
    return dw * s, (count + 2) * U * mag * abs(s) * (1 + HALF[dt]) + HALF[dt] * np.abs(dw * s) + TINY[dt] * (count > 0)


# ── linear cross entropy ──────────────────────────────────────────────────

def _product(a, b, dt, ea=0.0):
    """a @ b for operands of the type, a off by ea, and its error: the terms of
    an f32 sum. f32 operands are two f16 values each: hi + lo is off by half a
    step of lo, 2^-23 = 2u of the value, and lo lo (up to 2^-24 = u) is left
    out: 5u more of each term; and where lo is a subnormal number by half of
    2^-24 at a scale whose largest value is 2^14 at least, 2^-39 of it."""
    mag = (np.abs(a) + ea) @ np.abs(b)
    e = (a.shape[1] + 8) * U * mag
    if np.ndim(ea):
        e = e + ea @ np.abs(b)
    if dt == abi.F32:
        low = 2.0 ** -39
        e = e + low * (np.abs(a).max(initial=0.0) * np.abs(b).sum(0) + np.abs(b).max(initial=0.0) * np.abs(a).sum(1)[:, None])
    return a @ b, e


def _logits(x, w, dt):
    return _product(x, w.T, dt)


def _lse(z, ez):
    m = z.max(1, keepdims=True)
    s = np.exp(z - m)
    total = s.sum(1, keepdims=True)
    lse = (m + np.log(total))[:, 0]
    # exp: four roundings and those of its argument, (z - m) log2 e; the sum:
    # at most vocab / 64 values of a lane, and 64 steps more.
    rel = ((ez + 4 * U * (1 + np.abs(z - m))) * s).sum(1) / total[:, 0] + (z.shape[1] // 64 + 64) * U
    return lse, rel + 3 * U * np.abs(lse)


def cross_entropy(x, w, t, dt):
    """[(loss, bound), (lse, bound)]."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    z, ez = _logits(x, w, dt)
    lse, el = _lse(z, ez)
    on = (t >= 0) & (t < len(w))
    at = np.where(on, t, 0)
    zt, et = z[np.arange(len(t)), at], ez[np.arange(len(t)), at]
    return [(np.where(on, lse - zt, 0.0), np.where(on, el + et + 2 * U * (np.abs(lse) + np.abs(zt)), 0.0)), (lse, el)]


def cross_entropy_vjp(x, w, t, dloss, dt):
    """[(dx, bound), (dw, bound)] with the kernel's own lse. What rows without a
    target hold does not enter (zeros here)."""
    x, w, g = (np.asarray(a, np.float64) for a in (x, w, dloss))
    x = np.where(((t >= 0) & (t < len(w)))[:, None], x, 0.0)
    z, ez = _logits(x, w, dt)
    lse, el = _lse(z, ez)
    on = (t >= 0) & (t < len(w))
    p = np.exp(z - lse[:, None])
    ep = p * (ez + el[:, None] + 8 * U * (1 + np.abs(z) + np.abs(lse)[:, None]))
    p[np.arange(len(t))[on], t[on]] -= 1
    # exp of less than -87.3 is below 2^-126 and may be 0 in f32: 64 bits still
    # hold e^-700, so a difference of all of such a probability is no error.
    ep += 2 * U * np.abs(p) + NORMAL
    gg = np.where(on, g, 0.0)[:, None]
    xx = np.where(on[:, None], x, 0.0)
    ds, eds = p * gg, (ep + 2 * U * np.abs(p)) * np.abs(gg)
    # dS is stored in 16 bits, f32's in two f16 values (_product); both f16 forms
    # scaled, so that half the smallest step is 2^-39 of the largest dloss.
    if dt != abi.F32:
        eds = eds * (1 + HALF[dt]) + HALF[dt] * np.abs(ds)
    eds = eds + 2.0 ** -39 * np.abs(g[on]).max(initial=0.0)
    out = []
    for a, ea, m in ((ds, eds, w), (ds.T, eds.T, xx)):
        v, b = _product(a, m, dt, ea)
        out.append((v, b * (1 + HALF[dt]) + HALF[dt] * np.abs(v) + TINY[dt]))
    return out
