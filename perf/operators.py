"""Timed cases of the operators at a language model's two ends and between its
blocks: the embedding lookup with its gradient, layer norm with weight and bias
and their gradients, and the cross entropy of an output projection over a
vocabulary with the gradients of both its operands.

``run`` computes them in their plain form (elementary torch operations in 32
bits, rounded once) unless ``own`` is set; then it makes the framework's calls.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def listed():
    return [
        # Scoring one new token of each of 8 sequences (log-probabilities while
        # serving): forward only, the weight matrix is read once.
        {"name": "ce_score_rows8", "kind": "ce", "dtype": "bf16", "rows": 8, "dim": 768, "vocab": 32000,
         "train": False, "ignored": 0.0},
        # One training step's loss of 4 sequences x 512 positions, in the lazy
        # streams' own type and in bf16.
        {"name": "ce_train_f32", "kind": "ce", "dtype": "f32", "rows": 2048, "dim": 1024, "vocab": 32000,
         "train": True, "ignored": 0.0},
        {"name": "ce_train_bf16", "kind": "ce", "dtype": "bf16", "rows": 2048, "dim": 1024, "vocab": 32000,
         "train": True, "ignored": 0.0},
        # A large batch over a larger vocabulary, whose logits would take 1.6 GB.
        {"name": "ce_train_large", "kind": "ce", "dtype": "bf16", "rows": 8192, "dim": 2048, "vocab": 50257,
         "train": True, "ignored": 0.0},
        # Ragged everywhere, and a third of the positions (the prompts of a
        # tuning set) without a target.
        {"name": "ce_train_odd", "kind": "ce", "dtype": "f16", "rows": 1000, "dim": 777, "vocab": 32003,
         "train": True, "ignored": 0.3},
        # The embedding of a decoding step of 8 sequences: launch latency.
        {"name": "embed_rows8", "kind": "embed", "dtype": "f32", "tokens": 8, "dim": 768, "vocab": 32000,
         "train": False},
        # The same training step's embedding, forward and gradient.
        {"name": "embed_train_f32", "kind": "embed", "dtype": "f32", "tokens": 2048, "dim": 1024, "vocab": 32000,
         "train": True},
        # Many tokens: words as frequent as in a text, so one row of the
        # gradient sums thousands of them.
        {"name": "embed_train_long", "kind": "embed", "dtype": "bf16", "tokens": 65536, "dim": 1024,
         "vocab": 50257, "train": True},
        {"name": "embed_train_odd", "kind": "embed", "dtype": "f16", "tokens": 1537, "dim": 777, "vocab": 32003,
         "train": True},
        # Layer norm forward and backward: the benchmark's size, a training
        # step's of 4 x 512 positions, and ragged rows.
        {"name": "ln_train_4096", "kind": "ln", "dtype": "f32", "rows": 4096, "cols": 4096, "train": True},
        {"name": "ln_train_block", "kind": "ln", "dtype": "bf16", "rows": 2048, "cols": 1024, "train": True},
        {"name": "ln_train_odd", "kind": "ln", "dtype": "f16", "rows": 1000, "cols": 777, "train": True},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """As _log, half of them rounded to a multiple of 64 where large."""
    n = _log(rng, lo, hi)
    return max(64, n // 64 * 64) if n >= 64 and rng.random() < 0.5 else n


def draw(rng):
    kind = rng.choices(("ce", "embed", "ln"), (4, 3, 3))[0]
    dtype = rng.choice(("f32", "bf16", "f16"))
    while True:
        if kind == "ce":
            c = {"kind": "ce", "dtype": dtype, "rows": _size(rng, 1, 8192), "dim": _size(rng, 64, 2048),
                 "vocab": _size(rng, 1000, 50257), "train": rng.random() < 0.7,
                 "ignored": rng.choice((0.0, 0.0, 0.3))}
            # f32 products cost about six times the 16-bit ones.
            if work(c)["flops"] * (6 if dtype == "f32" else 1) <= 5e12:
                return c
        elif kind == "embed":
            c = {"kind": "embed", "dtype": dtype, "tokens": _log(rng, 1, 65536), "dim": _size(rng, 16, 4096),
                 "vocab": _size(rng, 250, 131072), "train": rng.random() < 0.7}
            if work(c)["bytes"] <= 4.7e8:
                return c
        else:
            c = {"kind": "ln", "dtype": dtype, "rows": _log(rng, 1, 16384), "cols": _size(rng, 16, 16384),
                 "train": rng.random() < 0.7}
            if c["rows"] * c["cols"] <= 1 << 24:
                return c


# ── inputs ────────────────────────────────────────────────────────────────

def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _words(gen, n, vocab):
    """Token ids about as frequent as words in a text: P(id) ~ 1 / (id + 1)."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)) - 1).long().clamp(0, vocab - 1).int()


def _params(case, seed):
    """Inputs of a case on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "ce":
        r, d, v = case["rows"], case["dim"], case["vocab"]
        # Logits of about unit spread, the target's raised by 0 to 16: rows
        # from unlearned to certain.
        w = _normal(g, (v, d), dt, 1 / math.sqrt(d))
        t = _words(g, r, v)
        lift = 16 * torch.rand((r, 1), generator=g, device="cuda")
        x = (torch.randn((r, d), generator=g, device="cuda") + lift * w[t.long()].float()).to(dt)
        skip = int(r * case["ignored"])
        t[:skip] = -100
        p = {"x": x, "w": w, "targets": t}
        if case["train"]:  # the mean's gradient; f16 trains with a loss scale
            p["dloss"] = torch.full((r,), (1024.0 if case["dtype"] == "f16" else 1.0) / max(1, r - skip), device="cuda")
        return p
    if case["kind"] == "embed":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        p = {"w": _normal(g, (v, d), dt, 1 / math.sqrt(d)), "ids": _words(g, n, v)}
        if case["train"]:
            p["dy"] = _normal(g, (n, d), dt)
        return p
    r, n = case["rows"], case["cols"]
    p = {"x": (torch.randn((r, n), generator=g, device="cuda") * 2 + 0.5).to(dt),
         "w": (1 + 0.2 * torch.randn(n, generator=g, device="cuda")).to(dt), "b": _normal(g, (n,), dt, 0.2)}
    if case["train"]:
        p["dy"] = _normal(g, (r, n), dt)
    return p


def prepare(case, seed):
    """Inputs and the buffers of the outputs."""
    s = {"case": case, **_params(case, seed)}
    if case["kind"] == "ce":
        s["loss"], s["lse"] = (torch.empty(case["rows"], device="cuda") for _ in range(2))
        outs = {"dx": "x", "dw": "w"}
    elif case["kind"] == "embed":
        s["y"] = torch.empty((case["tokens"], case["dim"]), dtype=DTYPES[case["dtype"]], device="cuda")
        outs = {"dw": "w"}
    else:
        s["y"] = torch.empty_like(s["x"])
        outs = {"dx": "x", "dw": "w", "db": "b"}
    if case["train"]:
        s.update({k: torch.empty_like(s[v]) for k, v in outs.items()})
    return s


# ── one pass ──────────────────────────────────────────────────────────────

def _own_ce(c, s):
    from oxidizedmlx_amd import abi, backend as hb
    dt = {"f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}[c["dtype"]]
    size = c["rows"], c["dim"], c["vocab"]
    x, w, t = s["x"].data_ptr(), s["w"].data_ptr(), s["targets"].data_ptr()
    hb.linear_cross_entropy(dt, x, w, t, s["loss"].data_ptr(), s["lse"].data_ptr(), *size)
    if not c["train"]:
        return {k: s[k] for k in ("loss", "lse")}
    hb.linear_cross_entropy_vjp(dt, x, w, t, s["lse"].data_ptr(), s["dloss"].data_ptr(), s["dx"].data_ptr(),
                                s["dw"].data_ptr(), *size)
    return {k: s[k] for k in ("loss", "lse", "dx", "dw")}


def _own_embed(c, s):
    from oxidizedmlx_amd import abi, backend as hb
    dt = {"f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}[c["dtype"]]
    size, scale = (c["tokens"], c["vocab"], c["dim"]), math.sqrt(c["dim"])
    hb.embedding_rows(dt, s["w"].data_ptr(), s["ids"].data_ptr(), s["y"].data_ptr(), *size, scale)
    if not c["train"]:
        return {"y": s["y"]}
    hb.embedding_vjp_rows(dt, s["dy"].data_ptr(), s["ids"].data_ptr(), s["dw"].data_ptr(), *size, scale)
    return {k: s[k] for k in ("y", "dw")}


def _own_ln(c, s):
    from oxidizedmlx_amd import abi, backend as hb
    dt = {"f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}[c["dtype"]]
    size = c["rows"], c["cols"], EPS
    x, w = s["x"].data_ptr(), s["w"].data_ptr()
    hb.layernorm_affine_rows(dt, x, w, s["b"].data_ptr(), s["y"].data_ptr(), *size)
    if not c["train"]:
        return {"y": s["y"]}
    hb.layernorm_affine_vjp_rows(dt, s["dy"].data_ptr(), x, w, s["dx"].data_ptr(), s["dw"].data_ptr(),
                                 s["db"].data_ptr(), *size)
    return {k: s[k] for k in ("y", "dx", "dw", "db")}


def _plain_ce(c, s):
    x, w, t = s["x"].float(), s["w"].float(), s["targets"].long()
    valid = (t >= 0) & (t < c["vocab"])
    at = torch.where(valid, t, 0)[:, None]
    z = x @ w.T
    m = z.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
    loss = torch.where(valid, (lse - z.gather(1, at))[:, 0], 0.0)
    out = {"loss": loss, "lse": lse[:, 0]}
    if not c["train"]:
        return out
    p = torch.exp(z - lse)
    p.scatter_add_(1, at, torch.full_like(lse, -1.0))
    p *= torch.where(valid, s["dloss"], 0.0)[:, None]
    return {**out, "dx": (p @ w).to(s["x"].dtype), "dw": (p.T @ x).to(s["w"].dtype)}


def _plain_embed(c, s):
    ids, scale = s["ids"].long().clamp(0, c["vocab"] - 1), math.sqrt(c["dim"])
    y = (s["w"][ids].float() * scale).to(s["w"].dtype)
    if not c["train"]:
        return {"y": y}
    dw = torch.zeros(s["w"].shape, device="cuda").index_add_(0, ids, s["dy"].float() * scale)
    return {"y": y, "dw": dw.to(s["w"].dtype)}


def _plain_ln(c, s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    xc = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(xc.square().mean(1, keepdim=True) + EPS)
    xh = xc * rstd
    y = (xh * w + b).to(s["x"].dtype)
    if not c["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    out = {"dx": dx, "dw": (dy * xh).sum(0), "db": dy.sum(0)}
    return {"y": y, **{k: v.to(s["x"].dtype) for k, v in out.items()}}


def run(state):
    c = state["case"]
    if own:
        return {"ce": _own_ce, "embed": _own_embed, "ln": _own_ln}[c["kind"]](c, state)
    return {"ce": _plain_ce, "embed": _plain_embed, "ln": _plain_ln}[c["kind"]](c, state)


# ── what a pass cannot do without ─────────────────────────────────────────

def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "ce":
        r, d, v = c["rows"], c["dim"], c["vocab"]
        # The operands in, the row results out, and in training the operands'
        # gradients; products of the logits and of the two gradients.
        n = (r + v) * d * size
        return {"bytes": n + 12 * r + ((n + 4 * r) if c["train"] else 0), "flops": (6 if c["train"] else 2) * r * d * v}
    if c["kind"] == "embed":
        n, d, v = c["tokens"], c["dim"], c["vocab"]
        # At most every token's row of the weight, each of the vocabulary's
        # rows once; the gradient is written whole.
        rows = min(n, v)
        return {"bytes": 4 * n + (rows + n) * d * size + ((4 * n + (n + v) * d * size) if c["train"] else 0), "flops": 0}
    r, n = c["rows"], c["cols"]
    return {"bytes": (2 * r * n + 2 * n) * size + (((3 * r * n + 3 * n) * size) if c["train"] else 0), "flops": 0}


# ── the same in 64 bits ───────────────────────────────────────────────────

def _exact_ce(c, p):
    x, w = p["x"].double(), p["w"].double()
    t = p["targets"].long()
    keep = torch.nonzero((t >= 0) & (t < c["vocab"]))[:, 0]
    lse = torch.empty(c["rows"], dtype=torch.float64, device="cuda")
    loss = torch.zeros_like(lse)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for lo in range(0, c["rows"], 1024):  # bounded memory
        lse[lo:lo + 1024] = torch.logsumexp(x[lo:lo + 1024] @ w.T, 1)
    for lo in range(0, len(keep), 1024):
        i = keep[lo:lo + 1024]
        z = x[i] @ w.T
        loss[i] = torch.nn.functional.cross_entropy(z, t[i], reduction="none")
        if c["train"]:
            q = torch.softmax(z, 1)
            q[torch.arange(len(i), device="cuda"), t[i]] -= 1
            q *= p["dloss"][i].double()[:, None]
            dx[i] = q @ w
            dw += q.T @ x[i]
    return {"loss": loss, "lse": lse, **({"dx": dx, "dw": dw} if c["train"] else {})}


def exact(case, seed):
    c, p = case, _params(case, seed)
    if c["kind"] == "ce":
        return _exact_ce(c, p)
    if c["kind"] == "embed":
        w = p["w"].double().requires_grad_(c["train"])
        y = torch.nn.functional.embedding(p["ids"].long().clamp(0, c["vocab"] - 1), w) * math.sqrt(c["dim"])
        if not c["train"]:
            return {"y": y}
        return {"y": y.detach(), "dw": torch.autograd.grad(y, w, p["dy"].double())[0]}
    leaves = [p[k].double().requires_grad_(c["train"]) for k in "xwb"]
    y = torch.nn.functional.layer_norm(leaves[0], (c["cols"],), leaves[1], leaves[2], EPS)
    if not c["train"]:
        return {"y": y}
    return {"y": y.detach(), **dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, p["dy"].double())))}
