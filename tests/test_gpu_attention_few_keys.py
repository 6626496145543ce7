"""Gradients of rows that see few keys: in 16-bit types those that see up to 64 have P
and dS in two terms and rowsum(dO o O) formed anew, whatever the heads' grouping and
the kernels' tiles. The bounds are attention_ref.attend_vjp's without what a single
rounding of P, dS and o may cost there."""
import numpy as np
import pytest

import attention_ref as A
import operators_ref as R
from operators_ref import HALF, TINY, U
from oxidizedmlx_amd import abi
from oxidizedmlx_amd import backend as hb
from test_gpu_packed_attention import Call, inputs, plan  # noqa: F401 (a fixture)

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

FEW = 64
TYPES = [abi.BF16, abi.F16]


def head_vjp(q, k, v, do, scale, causal, dt):
    """One head of a sequence: [(dq, e), (dk, e), (dv, e)] before the results' rounding."""
    n, d = q.shape
    o, eo, lse, el = A.attend(q, k, v, 0, scale, causal, dt)
    z, ez = A._scores(q, k, scale)
    seen = np.tril(np.ones((n, n), bool)) if causal else np.ones((n, n), bool)
    few = seen.sum(1, keepdims=True) <= FEW
    p = np.where(seen, np.exp(z - lse[:, None]), 0.0)
    rel = ez + el[:, None] + 6 * U * (2 + np.abs(z) + np.abs(lse)[:, None])
    ado, av, aq, ak = np.abs(do), np.abs(v), np.abs(q), np.abs(k)
    dp, edp = do @ v.T, (d + 8) * U * (ado @ av.T)
    delta = (do * o).sum(1, keepdims=True)
    rounded = (ado * eo).sum(1, keepdims=True) + (d + 8) * U * (ado * np.abs(o)).sum(1, keepdims=True)
    # Formed anew: D0 + sum of P (dP - D0) for a D0 that is off by `rounded`, which a P whose sum is 1 takes
    # out again. What is left: P's and dP's errors, the sum over the keys, two steps of D itself.
    size = np.abs(dp) + np.abs(delta) + rounded
    anew = (p * (rel * size + edp + (n + 16) * U * size)).sum(1, keepdims=True) + 2 * U * (np.abs(delta) + rounded)
    edelta = np.where(few, anew, rounded)
    # A value in two terms is off by half a step of the second, which is half a step of the first at most.
    step = np.where(few, HALF[dt] ** 2, HALF[dt])
    ds = p * (dp - delta)
    eds = np.abs(ds) * (rel + 4 * U + step) + p * (1 + rel + step) * (edp + edelta + 2 * U * (np.abs(dp) + np.abs(delta)))
    # f16: half the smallest step, 2^-25, where the largest of a column is 2^12 (of dS) or 1 is 2^14 (of P).
    eds_q, eds_k = (eds + 2.0 ** -36 * np.abs(ds).max(a, keepdims=True) * seen for a in (1, 0))
    s, terms = abs(scale), (2 * n + 8) * U
    return [(scale * ds @ k, s * (eds_q @ ak + terms * (np.abs(ds) @ ak))),
            (scale * ds.T @ q, s * (eds_k.T @ aq + terms * (np.abs(ds).T @ aq))),
            (p.T @ do, (p * (rel + step)).T @ ado + terms * (p.T @ ado) + 2.0 ** -39 * seen.T @ ado)]


def packed_vjp(q, k, v, do, starts, scale, causal, dt):
    q, k, v, do = (np.asarray(t, np.float64) for t in (q, k, v, do))
    group = q.shape[1] // k.shape[1]
    vals, errs = [np.zeros(t.shape) for t in (q, k, v)], [np.zeros(t.shape) for t in (q, k, v)]
    for a, b in zip(starts, starts[1:]):
        for h in range(q.shape[1]):
            g = h // group
            for i, (x, e) in enumerate(head_vjp(q[a:b, h], k[a:b, g], v[a:b, g], do[a:b, h], scale, causal, dt)):
                at = g if i else h
                vals[i][a:b, at] += x
                errs[i][a:b, at] += e + (group * U * np.abs(x) if i else 0)
    return [(x, e * (1 + HALF[dt]) + (HALF[dt] + 4 * U) * np.abs(x) + TINY[dt]) for x, e in zip(vals, errs)]


def gradients(q, k, v, do, starts, scale, causal, dt):
    c = Call(q, k, v, do, starts, dt)
    c.forward(scale, causal)
    c.backward(scale, causal)
    hb.synchronize()
    return c.results()[2:]


# heads of one, three, four and five to a K/V head; sequences that end in, at and past the 64th token
@pytest.mark.parametrize("dt", TYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("heads,kv", [(2, 2), (3, 1), (4, 1), (5, 1)])
@pytest.mark.parametrize("tokens,dim,starts,causal", [(300, 64, [0, 300], True), (330, 128, [0, 63, 127, 192, 330], True),
                                                      (200, 40, [0, 130, 200], True), (150, 128, [0, 64, 87, 150], False)])
def test_matches_64_bits(tokens, dim, starts, causal, heads, kv, dt, plan):  # noqa: F811
    print(f"few keys {tokens} {heads}/{kv} {dim} {starts} causal {causal} {R.NAMES[dt]}", flush=True)
    data, scale = inputs(tokens, heads, kv, dim, dt, seed=dim), dim ** -0.5
    wants = packed_vjp(*data, starts, scale, causal, dt)
    for name, got, (want, bound) in zip(("dq", "dk", "dv"), gradients(*data, starts, scale, causal, dt), wants):
        R.check(got, want, bound, name)
