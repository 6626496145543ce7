"""64-bit forms of rotary positions, attention of packed sequences with grouped
heads, its gradient, and attention over a cache in pages, with the error bounds of
their kernels (U, HALF, TINY and check of operators_ref).

A score is a sum of dim products in f32; p = exp(score - max) takes it, the factor
scale log2 e rounded twice, the difference's rounding and exp2's; p is rounded
to the operands' type for its product (f16 holds it times 2^6 or more: what is lost
below is 2^-31 of the row's largest)."""
import numpy as np

import operators_ref as R
from operators_ref import HALF, TINY, U

# What rounding p or dS to the operands' type may lose: f32 rounds nothing.
STEP = {dt: (0.0 if h == U else h) for dt, h in HALF.items()}
FLOOR = 2.0 ** -31


def rope(x, positions, freqs, rotary, interleaved, magnitude, dt, sign=1.0):
    """x [tokens, heads, dim] turned, and its bound."""
    x = np.asarray(x, np.float64)
    a = np.asarray(positions, np.float64)[:, None] * freqs
    c, s = (magnitude * f(a)[:, None] for f in (np.cos, np.sin))
    s = s * sign
    at = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    u, v = x[..., at[0]], x[..., at[1]]
    y, e = x.copy(), np.zeros_like(x)
    y[..., at[0]], y[..., at[1]] = u * c - v * s, v * c + u * s
    # The angle is rounded at an eighth of a turn, 2^-25 radians; cosine and sine are off
    # by two steps, times the magnitude one rounding, two products and a sum; angles of
    # far positions by 2^-50 of themselves.
    off = (2 * U + 8 * U + np.abs(a)[:, None] * 2.0 ** -50) * abs(magnitude) * (np.abs(u) + np.abs(v))
    e[..., at[0]] = e[..., at[1]] = off
    turned = np.zeros(x.shape[-1], bool)
    turned[:rotary] = True
    return y, np.where(turned, e * (1 + HALF[dt]) + HALF[dt] * np.abs(y) + TINY[dt], 0.0)


def _scores(q, k, scale):
    z = scale * (q @ k.T)
    # dim products summed, the factor c (two roundings), its product.
    return z, (q.shape[1] + 8) * U * abs(scale) * (np.abs(q) @ np.abs(k).T) + 4 * U * np.abs(z)


def attend(q, k, v, first, scale, causal, dt):
    """One head: rows q from position first over keys k, v. (o, eo, lse, el)."""
    m, n = len(q), len(k)
    z, ez = _scores(q, k, scale)
    seen = np.arange(n)[None, :] <= (first + np.arange(m))[:, None] if causal else np.ones((m, n), bool)
    none = ~seen.any(1)
    z = np.where(seen, z, -np.inf)
    top = np.where(none, 0.0, z.max(1, initial=-np.inf))[:, None]
    e = np.exp(z - top)
    total = e.sum(1, keepdims=True)
    p = e / np.where(total == 0, 1.0, total)
    rel = np.where(seen, ez + 4 * U * (2 + np.abs(np.where(seen, z, 0.0)) + np.abs(top)), 0.0)
    # A lane sums half of the keys; the halves, the waves and the parts join: 80 more.
    rl = (p * rel).sum(1, keepdims=True) + (n / 2 + 80) * U
    av = np.abs(v)
    # o: p's error and rounding, the sum over n keys (the parts' joins 80 more), the division.
    eo = (p * (rel + rl + STEP[dt])) @ av + (n + 88) * U * (p @ av) + (FLOOR * seen @ av if STEP[dt] else 0.0)
    o = p @ v
    with np.errstate(divide="ignore"):
        lse = (top + np.log(total))[:, 0]
    el = rl[:, 0] + 4 * U * (1 + np.abs(top[:, 0]) + np.abs(np.where(none, 0.0, lse)))
    return o, eo * (1 + HALF[dt]) + HALF[dt] * np.abs(o) + TINY[dt], np.where(none, -np.inf, lse), el


def attend_vjp(q, k, v, do, scale, causal, dt):
    """One head of a sequence: [(dq, e), (dk, e), (dv, e)] for the forward's own o
    and lse, before the results' rounding."""
    n, d = q.shape
    o, eo, lse, el = attend(q, k, v, 0, scale, causal, dt)
    z, ez = _scores(q, k, scale)
    seen = np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool)
    p = np.where(seen, np.exp(z - lse[:, None]), 0.0)
    rel = ez + el[:, None] + 6 * U * (2 + np.abs(z) + np.abs(lse)[:, None])
    ado, av, aq, ak = np.abs(do), np.abs(v), np.abs(q), np.abs(k)
    dp, edp = do @ v.T, (d + 8) * U * (ado @ av.T)
    delta = (do * o).sum(1, keepdims=True)
    edelta = (ado * eo).sum(1, keepdims=True) + (d + 8) * U * (ado * np.abs(o)).sum(1, keepdims=True)
    ds = p * (dp - delta)
    eds = np.abs(ds) * (rel + 4 * U + STEP[dt]) + p * (1 + rel + STEP[dt]) * (edp + edelta + 2 * U * (np.abs(dp) + np.abs(delta)))
    if STEP[dt]:  # f16: 2^-36 of the largest of its column, rows for dq, keys for dk
        eds_q, eds_k = (eds + 2.0 ** -36 * np.abs(ds).max(a, keepdims=True) * seen for a in (1, 0))
    else:
        eds_q = eds_k = eds
    s = abs(scale)
    out = [(scale * ds @ k, s * (eds_q @ ak + (n + 8) * U * (np.abs(ds) @ ak))),
           (scale * ds.T @ q, s * (eds_k.T @ aq + (n + 8) * U * (np.abs(ds).T @ aq))),
           (p.T @ do, (p * (rel + STEP[dt])).T @ ado + (n + 8) * U * (p.T @ ado) + (2.0 ** -39 * seen.T @ ado if STEP[dt] else 0))]
    return out


def packed(q, k, v, starts, scale, causal, dt):
    """q [tokens, heads, dim], k and v [tokens, kv_heads, dim]: (o, eo, lse, el);
    NaN where no sequence is."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    o, eo = np.full(q.shape, np.nan), np.zeros(q.shape)
    lse, el = np.full(q.shape[:2], np.nan), np.zeros(q.shape[:2])
    group = q.shape[1] // k.shape[1]
    for a, b in zip(starts, starts[1:]):
        for h in range(q.shape[1] if b > a else 0):
            g = h // group
            o[a:b, h], eo[a:b, h], lse[a:b, h], el[a:b, h] = attend(q[a:b, h], k[a:b, g], v[a:b, g], 0, scale, causal, dt)
    return o, eo, lse, el


def packed_vjp(q, k, v, do, starts, scale, causal, dt):
    """[(dq, e), (dk, e), (dv, e)]; NaN where no sequence is."""
    q, k, v, do = (np.asarray(t, np.float64) for t in (q, k, v, do))
    group = q.shape[1] // k.shape[1]
    vals, errs = [np.full(t.shape, np.nan) for t in (q, k, v)], [np.zeros(t.shape) for t in (q, k, v)]
    for a, b in zip(starts, starts[1:]):
        for i in (1, 2):
            vals[i][a:b] = 0
        for h in range(q.shape[1] if b > a else 0):
            g = h // group
            parts = attend_vjp(q[a:b, h], k[a:b, g], v[a:b, g], do[a:b, h], scale, causal, dt)
            for i, (x, e) in enumerate(parts):
                at = h if i == 0 else g
                vals[i][a:b, at] = x if i == 0 else vals[i][a:b, at] + x
                errs[i][a:b, at] += e + (group * U * np.abs(x) if i else 0)
    return [(x, e * (1 + HALF[dt]) + (HALF[dt] + 4 * U) * np.abs(x) + TINY[dt]) for x, e in zip(vals, errs)]


def pages_of(seqs, page, table_width, pages, rng):
    """The table: page numbers in no order for sequences of these lengths."""
    order = rng.permutation(pages)
    table, at = np.full((len(seqs), table_width), -7, np.int32), 0
    for i, n in enumerate(seqs):
        c = -(-n // page)
        table[i, :c] = order[at:at + c]
        at += c
    return table


def same_where(got, want, bound, what):
    """R.check where a sequence is (want is not NaN); returns the mask of the rest."""
    on = ~np.isnan(want)
    R.check(got[on], want[on], np.broadcast_to(bound, want.shape)[on], what)
    return ~on
