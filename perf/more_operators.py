"""Timed cases of a transformer's attention over several sequences at once:
rotary positions with their gradient, causal attention of packed sequences with
grouped heads and its gradient, a cache in pages that new tokens are appended
to, and the attention of new tokens over it.

``run`` computes them in their plain form (elementary torch operations in 32
bits, angles in 64, rounded once) unless ``own`` is set; then it makes the
framework's calls.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BASE = 10000.0


def listed():
    return [
        # Queries of a decoding step of 8 sequences, rotated: launch latency.
        {"name": "rope_step", "kind": "rope", "dtype": "f32", "tokens": 8, "heads": 12, "dim": 64, "rotary": 64,
         "interleaved": False, "factor": 1.0, "far": 144, "train": False},
        # Queries and keys of a training step on long texts, their positions
        # scaled: forward and gradient.
        {"name": "rope_train_long", "kind": "rope", "dtype": "bf16", "tokens": 16384, "heads": 40, "dim": 128,
         "rotary": 128, "interleaved": False, "factor": 8.0, "far": 131072, "train": True},
        # The keys and values of one token of each of 64 sequences into a cache.
        {"name": "append_step", "kind": "append", "dtype": "bf16", "seqs": 64, "new": 64, "len": 4096, "kv_heads": 8,
         "dim": 128, "page": 16, "rotary": 128, "interleaved": False},
        # Prompts into a cache: ragged, part of the head rotated, in pairs.
        {"name": "append_prompts", "kind": "append", "dtype": "f16", "seqs": 7, "new": 5001, "len": 8192, "kv_heads": 5,
         "dim": 80, "page": 64, "rotary": 40, "interleaved": True},
        # A training step's block of 4 sequences of 512 in the lazy streams' own type.
        {"name": "packed_block_f32", "kind": "packed", "dtype": "f32", "seqs": 4, "tokens": 2048, "even": True,
         "heads": 16, "kv_heads": 16, "dim": 64, "causal": True, "train": True},
        # Texts of different lengths packed into one training step.
        {"name": "packed_train", "kind": "packed", "dtype": "bf16", "seqs": 6, "tokens": 8192, "even": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "causal": True, "train": True},
        # Ragged everywhere.
        {"name": "packed_odd", "kind": "packed", "dtype": "f16", "seqs": 5, "tokens": 1537, "even": False, "heads": 9,
         "kv_heads": 3, "dim": 80, "causal": True, "train": True},
        # One long prompt, forward only.
        {"name": "packed_prompt", "kind": "packed", "dtype": "bf16", "seqs": 1, "tokens": 32768, "even": True, "heads": 16,
         "kv_heads": 4, "dim": 128, "causal": True, "train": False},
        # A decoding step of 8 short sequences: latency.
        {"name": "paged_step", "kind": "paged", "dtype": "f32", "seqs": 8, "new": 8, "len": 144, "even": True, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16},
        # A decoding step of many sequences of different lengths.
        {"name": "paged_many", "kind": "paged", "dtype": "bf16", "seqs": 64, "new": 64, "len": 8192, "even": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16},
        # A decoding step of two very long sequences: few rows, many keys.
        {"name": "paged_long", "kind": "paged", "dtype": "f16", "seqs": 2, "new": 2, "len": 131072, "even": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # Chunks of prompts over what the cache holds of them.
        {"name": "paged_chunk", "kind": "paged", "dtype": "bf16", "seqs": 4, "new": 2000, "len": 16384, "even": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("rope", "append", "packed", "paged"), (2, 1, 4, 4))[0]
    dtype = rng.choice(("f32", "bf16", "f16"))
    while True:
        dim = rng.choice((64, 128, 8 * rng.randint(2, 16)))
        kv = rng.choice((1, 2, 4, 8, 8, rng.randint(1, 16)))
        heads = kv * rng.choice((1, 1, 2, 4, 4, 8, rng.randint(1, 8)))
        rotary = rng.choice((dim, dim, 2 * rng.randint(1, dim // 2)))
        c = {"kind": kind, "dtype": dtype}
        if kind == "rope":
            c.update(tokens=_log(rng, 1, 65536), heads=heads, dim=dim, rotary=rotary, interleaved=rng.random() < 0.4,
                     factor=rng.choice((1.0, 1.0, 4.0, 8.0)), far=_log(rng, 64, 1000000), train=rng.random() < 0.6)
            c["far"] = max(c["far"], c["tokens"])
            if work(c)["bytes"] <= 6.5e8:
                return c
            continue
        # f32 products run at a sixteenth of the 16-bit ones' rate.
        slow = 16 if dtype == "f32" else 1
        if kind == "packed":
            seqs = _log(rng, 1, 64)
            c.update(seqs=seqs, tokens=max(seqs, _log(rng, 16, 32768)), even=rng.random() < 0.3, heads=heads, kv_heads=kv,
                     dim=dim, causal=rng.random() < 0.85, train=rng.random() < 0.6)
            # The plain form's time goes by the scores, whole or causal.
            if work(c)["flops"] * slow <= 4.4e12 and work(c)["flops"] / dim * 128 <= 4.4e12:
                return c
            continue
        seqs = _log(rng, 1, 128)
        new = seqs * (1 if rng.random() < 0.5 else _log(rng, 1, 512))
        c.update(seqs=seqs, new=new, len=max(-(-new // seqs), _log(rng, 16, 131072)), kv_heads=kv, dim=dim,
                 page=rng.choice((16, 16, 32, 64, 128, 256)))
        if kind == "append":
            c.update(rotary=rotary, interleaved=rng.random() < 0.4)
            if seqs * c["len"] * kv * dim <= 1 << 27 and seqs * c["len"] >= new:
                return c
        else:
            c.update(even=rng.random() < 0.4, heads=heads)
            if seqs * c["len"] * kv * dim <= 1 << 28 and work(c)["flops"] * slow <= 1.1e12:
                return c


# ── lengths ───────────────────────────────────────────────────────────────

def _parts(total, n, even, rng):
    """total as n whole numbers of 1 and more, equal or spread over a factor of about 16."""
    weights = [1.0 if even else 2 ** (4 * rng.random()) for _ in range(n)]
    cuts, run = [0], 0.0
    for w in weights:
        run += w
        cuts.append(round(run / sum(weights) * (total - n)))
    return [b - a + 1 for a, b in zip(cuts, cuts[1:])]


def _lengths(c):
    """(new tokens, whole length) of each sequence: of the case alone."""
    rng = random.Random(c["seqs"] * 7919 + c["dim"])
    if c["kind"] == "packed":
        n = _parts(c["tokens"], c["seqs"], c["even"], rng)
        return n, n
    new = _parts(c["new"], c["seqs"], c["new"] == c["seqs"], rng)
    even = c.get("even", False)
    return new, [max(n, c["len"] if even or i == 0 else int(c["len"] * 2 ** (-4 * rng.random()))) for i, n in enumerate(new)]


def _frequencies(c):
    """f64 angles per position: base^(-2i/rotary), divided by the factor where a
    turn is longer than an original context of 8192 and not at all from 4 turns on."""
    i = torch.arange(c["rotary"] // 2, dtype=torch.float64, device="cuda")
    f = BASE ** (-2 * i / c["rotary"])
    if c.get("factor", 1.0) == 1.0:
        return f
    keep = ((f * 8192 / (2 * math.pi) - 1) / 3).clamp(0, 1)
    return f * (keep + (1 - keep) / c["factor"])


# ── inputs ────────────────────────────────────────────────────────────────

def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _starts(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _params(case, seed):
    """Inputs of a case on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]
    if c["kind"] == "rope":
        p = {"x": _normal(g, (c["tokens"], c["heads"], c["dim"]), dt),
             "positions": torch.randint(0, c["far"], (c["tokens"],), generator=g, device="cuda").int()}
        if c["train"]:
            p["dy"] = _normal(g, (c["tokens"], c["heads"], c["dim"]), dt)
        return p
    new, lens = _lengths(c)
    p = {"starts": _ints(_starts(new))}
    if c["kind"] == "packed":
        # Queries, keys and values as one projection writes them.
        row = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        p["qkv"] = _normal(g, (c["tokens"], row), dt)
        if c["train"]:
            p["dout"] = _normal(g, (c["tokens"], c["heads"], c["dim"]), dt)
        return p
    # Pages in no order, as a server that has been running hands them out.
    per = [-(-n // c["page"]) for n in lens]
    width = max(per)
    order = torch.randperm(sum(per) + 3, generator=g, device="cuda").int()
    p["table"] = torch.zeros((c["seqs"], width), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        p["table"][i, :n] = order[at:at + n]
        at += n
    p["lens"] = _ints(lens)
    pages = (sum(per) + 3, c["kv_heads"], c["page"], c["dim"])
    p["k_pages"], p["v_pages"] = _normal(g, pages, dt), _normal(g, pages, dt)
    if c["kind"] == "append":
        p["kv"] = _normal(g, (c["new"], 2, c["kv_heads"], c["dim"]), dt)
    else:
        p["q"] = _normal(g, (c["new"], c["heads"], c["dim"]), dt)
    return p


def prepare(case, seed):
    """Inputs, the table of frequencies and the buffers of the outputs."""
    c = case
    s = {"case": c, **_params(c, seed)}
    if "rotary" in c:
        s["freqs"] = _frequencies(c)
    if c["kind"] == "rope":
        s["y"] = torch.empty_like(s["x"])
        if c["train"]:
            s["dx"] = torch.empty_like(s["x"])
        return s
    s["new"], s["all"] = _lengths(c)
    if c["kind"] == "packed":
        s["o"] = torch.empty((c["tokens"], c["heads"], c["dim"]), dtype=s["qkv"].dtype, device="cuda")
        s["lse"] = torch.empty((c["tokens"], c["heads"]), device="cuda")
        if c["train"]:
            s["dqkv"] = torch.empty_like(s["qkv"])
    elif c["kind"] == "paged":
        s["o"] = torch.empty_like(s["q"])
    return s


# ── one pass: the framework's calls ───────────────────────────────────────

def _dtype(c):
    from oxidizedmlx_amd import abi
    return {"f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}[c["dtype"]]


def _own_rope(c, s):
    from oxidizedmlx_amd import backend as hb
    row = c["heads"] * c["dim"]
    args = c["tokens"], c["heads"], c["dim"], c["rotary"], row, row, c["interleaved"], 1.0
    pos, freqs = s["positions"].data_ptr(), s["freqs"].data_ptr()
    hb.rope_rows(_dtype(c), s["x"].data_ptr(), pos, freqs, s["y"].data_ptr(), *args)
    if not c["train"]:
        return {"y": s["y"]}
    hb.rope_vjp_rows(_dtype(c), s["dy"].data_ptr(), pos, freqs, s["dx"].data_ptr(), *args)
    return {"y": s["y"], "dx": s["dx"]}


def _split(c, t):
    """Query, key and value parts of a [tokens, row] projection or its gradient."""
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    return [v.unflatten(1, (-1, d)) for v in t.split((h * d, kv * d, kv * d), 1)]


def _own_packed(c, s):
    from oxidizedmlx_amd import backend as hb
    q, k, v = (t.data_ptr() for t in _split(c, s["qkv"]))
    row = s["qkv"].stride(0)
    args = (c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], row, row, c["heads"] * c["dim"],
            c["dim"] ** -0.5, c["causal"])
    starts, o, lse = (s[n].data_ptr() for n in ("starts", "o", "lse"))
    hb.packed_attention(_dtype(c), q, k, v, starts, o, lse, *args)
    if not c["train"]:
        return {"o": s["o"], "lse": s["lse"]}
    dq, dk, dv = _split(c, s["dqkv"])
    hb.packed_attention_vjp(_dtype(c), q, k, v, o, s["dout"].data_ptr(), lse, starts, dq.data_ptr(), dk.data_ptr(),
                            dv.data_ptr(), *args)
    return {"o": s["o"], "lse": s["lse"], "dq": dq, "dk": dk, "dv": dv}


def _pages(c, s):
    return s["k_pages"].shape[0], c["page"], s["table"].shape[1]


def _own_append(c, s):
    from oxidizedmlx_amd import backend as hb
    k, v = s["kv"].unbind(1)
    hb.paged_append(_dtype(c), k.data_ptr(), v.data_ptr(), s["starts"].data_ptr(), s["lens"].data_ptr(),
                    s["table"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), c["seqs"], c["new"],
                    c["kv_heads"], c["dim"], s["kv"].stride(0), *_pages(c, s), s["freqs"].data_ptr(), c["rotary"],
                    c["interleaved"], 1.0)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _own_paged(c, s):
    from oxidizedmlx_amd import backend as hb
    row = c["heads"] * c["dim"]
    hb.paged_attention(_dtype(c), s["q"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr(),
                       s["starts"].data_ptr(), s["lens"].data_ptr(), s["table"].data_ptr(), s["o"].data_ptr(), c["seqs"],
                       c["new"], c["heads"], c["kv_heads"], c["dim"], row, row, *_pages(c, s), c["dim"] ** -0.5)
    return {"o": s["o"]}


# ── one pass: plain ───────────────────────────────────────────────────────

def _rotate(c, x, positions, freqs, sign=1.0):
    """Rotated x [tokens, heads, dim] in 32 bits, angles in 64."""
    a = positions.double()[:, None] * freqs
    cos, sin = torch.cos(a).float()[:, None], (sign * torch.sin(a)).float()[:, None]
    out, r = x.float(), c["rotary"]
    at = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    u, v = (out[..., i] for i in at)
    y = out.clone()
    y[..., at[0]], y[..., at[1]] = u * cos - v * sin, v * cos + u * sin
    return y.to(x.dtype)


def _plain_rope(c, s):
    out = {"y": _rotate(c, s["x"], s["positions"], s["freqs"])}
    if c["train"]:
        out["dx"] = _rotate(c, s["dy"], s["positions"], s["freqs"], -1.0)
    return out


def _scores(c, q, k, first, causal):
    """Masked scores [kv_heads, group, rows, keys] of the queries from position
    first on, their heads grouped: [kv_heads, group, rows, dim]."""
    z = torch.matmul(q, k[:, None].transpose(2, 3).contiguous()) * c["dim"] ** -0.5
    if causal:
        rows = torch.arange(first, first + q.shape[2], device="cuda")[:, None]
        z.masked_fill_(torch.arange(k.shape[1], device="cuda") > rows, -math.inf)
    return z


def _step(c, keys):
    """Query rows at a time, so that the scores stay at 1 GiB."""
    return max(1, (1 << 28) // (c["heads"] * max(keys, 1)))


def _grouped(c, x):
    """[tokens, heads, dim] in 32 bits as [kv_heads, group, tokens, dim]."""
    return x.float().transpose(0, 1).unflatten(0, (c["kv_heads"], -1))


def _flat(x):
    return x.flatten(0, 1).transpose(0, 1)


def _attend(c, q, k, v, first, causal):
    """o [rows, heads, dim] and lse [rows, heads] in 32 bits."""
    q, k, v = _grouped(c, q), k.float().transpose(0, 1).contiguous(), v.float().transpose(0, 1).contiguous()
    n = k.shape[1]
    o, lse = [], []
    for lo in range(0, q.shape[2], _step(c, n)):
        hi = min(q.shape[2], lo + _step(c, n))
        end = min(n, first + hi) if causal else n
        z = _scores(c, q[:, :, lo:hi].contiguous(), k[:, :end], first + lo, causal)
        m = z.amax(3, keepdim=True)
        e = torch.exp(z - m)
        total = e.sum(3, keepdim=True)
        o.append(_flat(torch.matmul(e, v[:, None, :end]) / total))
        lse.append(_flat(m + torch.log(total))[..., 0])
    return torch.cat(o), torch.cat(lse)


def _attend_vjp(c, q, k, v, do, o, lse, causal):
    """dq [rows, heads, dim], dk and dv [rows, kv_heads, dim] in 32 bits."""
    q, do, o = (_grouped(c, t) for t in (q, do, o))
    lse = lse.transpose(0, 1).unflatten(0, (c["kv_heads"], -1))[..., None]
    k, v = (t.float().transpose(0, 1).contiguous() for t in (k, v))
    dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    delta, n, scale = (do * o).sum(3, keepdim=True), k.shape[1], c["dim"] ** -0.5
    for lo in range(0, n, _step(c, n)):
        hi = min(n, lo + _step(c, n))
        end = hi if causal else n
        qs, ds = q[:, :, lo:hi].contiguous(), do[:, :, lo:hi].contiguous()
        p = torch.exp(_scores(c, qs, k[:, :end], lo, causal) - lse[:, :, lo:hi])
        dv[:, :end] += torch.matmul(p.transpose(2, 3), ds).sum(1)
        t = p * (torch.matmul(ds, v[:, None, :end].transpose(2, 3).contiguous()) - delta[:, :, lo:hi]) * scale
        dq[:, :, lo:hi] = torch.matmul(t, k[:, None, :end])
        dk[:, :end] += torch.matmul(t.transpose(2, 3), qs).sum(1)
    return _flat(dq), dk.transpose(0, 1), dv.transpose(0, 1)


def _plain_packed(c, s):
    q, k, v = _split(c, s["qkv"])
    parts, at = [], 0
    for n in s["new"]:
        i = slice(at, at + n)
        at += n
        o, lse = _attend(c, q[i], k[i], v[i], 0, c["causal"])
        grads = _attend_vjp(c, q[i], k[i], v[i], s["dout"][i], o, lse, c["causal"]) if c["train"] else ()
        parts.append((o, lse, *grads))
    out = dict(zip(("o", "lse", "dq", "dk", "dv"), (torch.cat(t) for t in zip(*parts))))
    return {n: t if n == "lse" else t.to(s["qkv"].dtype) for n, t in out.items()}


def _plain_append(c, s):
    k, v = s["kv"].unbind(1)
    positions = torch.cat([torch.arange(n - m, n, device="cuda") for m, n in zip(s["new"], s["all"])])
    k = _rotate(c, k, positions, s["freqs"])
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), s["starts"].diff())
    page = s["table"][seq, positions // c["page"]].long()
    s["k_pages"][page, :, positions % c["page"]] = k
    s["v_pages"][page, :, positions % c["page"]] = v
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_paged(c, s):
    out, at = [], 0
    for i, (m, n) in enumerate(zip(s["new"], s["all"])):
        pages = s["table"][i, :-(-n // c["page"])].long()
        k, v = (s[t][pages].transpose(1, 2).flatten(0, 1)[:n] for t in ("k_pages", "v_pages"))
        out.append(_attend(c, s["q"][at:at + m], k, v, n - m, True)[0])
        at += m
    return {"o": torch.cat(out).to(s["q"].dtype)}


def run(state):
    c = state["case"]
    which = (_own_rope, _own_packed, _own_append, _own_paged) if own else (_plain_rope, _plain_packed, _plain_append,
                                                                          _plain_paged)
    return which[("rope", "packed", "append", "paged").index(c["kind"])](c, state)


# ── what a pass cannot do without ─────────────────────────────────────────

def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "rope":
        n = c["tokens"] * c["heads"] * c["dim"] * size
        return {"bytes": (2 * n + 4 * c["tokens"] + 4 * c["rotary"]) * (2 if c["train"] else 1), "flops": 0}
    new, lens = _lengths(c)
    if c["kind"] == "append":
        # Rows read and written, and a page number for each page they reach.
        return {"bytes": 4 * c["new"] * c["kv_heads"] * c["dim"] * size + 12 * c["seqs"]
                + 4 * sum(-(-m // c["page"]) for m in new), "flops": 0}
    rows = c["tokens"] if c["kind"] == "packed" else c["new"]
    q, kv = rows * c["heads"] * c["dim"] * size, sum(lens) * c["kv_heads"] * c["dim"] * size
    causal = c.get("causal", True)
    pairs = sum(m * n - m * (m - 1) // 2 if causal else m * n for m, n in zip(new, lens))
    flops = 4 * c["heads"] * c["dim"] * pairs
    if c["kind"] == "paged":
        return {"bytes": 2 * q + 2 * kv + 8 * c["seqs"] + 4 * sum(-(-n // c["page"]) for n in lens), "flops": flops}
    lse = 4 * rows * c["heads"]
    if not c["train"]:
        return {"bytes": 2 * q + 2 * kv + lse, "flops": flops}
    # The gradient reads q, k, v, o, its cotangent and lse, writes dq, dk and dv: five products of the pairs.
    return {"bytes": 6 * q + 6 * kv + 2 * lse, "flops": 7 * flops // 2}


# ── the same in 64 bits ───────────────────────────────────────────────────

def _turned(c, x, positions):
    """x as complex pairs times e^(i angle)."""
    x, r = x.double(), c["rotary"]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), positions.double()[:, None] * _frequencies(c))
    head = x[..., :r]
    pairs = head.unflatten(-1, (r // 2, 2)) if c["interleaved"] else torch.stack(head.split(r // 2, -1), -1)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
    back = z.flatten(-2) if c["interleaved"] else torch.cat(z.unbind(-1), -1)
    return torch.cat((back, x[..., r:]), -1)


def _exact_rows(c, q, k, v, mask, scale):
    """o and lse of one head's rows [n, dim]."""
    z = (q @ k.T) * scale
    if mask is not None:
        z = z.masked_fill(mask, -math.inf)
    return torch.softmax(z, 1) @ v, torch.logsumexp(z, 1)


def _exact_head(c, q, k, v, first, causal, rows=4096):
    o, lse = [], []
    for lo in range(0, len(q), rows):
        part = q[lo:lo + rows]
        mask = None
        if causal:
            mask = torch.ones((len(part), len(k)), dtype=torch.bool, device="cuda").triu(first + lo + 1)
        y, z = _exact_rows(c, part, k, v, mask, 1 / math.sqrt(c["dim"]))
        o.append(y)
        lse.append(z)
    return torch.cat(o), torch.cat(lse)


def _exact_packed(c, p):
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    x = p["qkv"].double()
    out = {"o": torch.empty((c["tokens"], h, d), dtype=torch.float64, device="cuda"),
           "lse": torch.empty((c["tokens"], h), dtype=torch.float64, device="cuda")}
    if c["train"]:
        out.update(dq=torch.empty_like(out["o"]), dk=torch.zeros((c["tokens"], kv, d), dtype=torch.float64, device="cuda"),
                   dv=torch.zeros((c["tokens"], kv, d), dtype=torch.float64, device="cuda"))
    at = 0
    for n in _lengths(c)[0]:
        i = slice(at, at + n)
        at += n
        for head in range(h):
            g = head * kv // h
            leaves = [x[i, lo:lo + d].clone().requires_grad_(c["train"])
                      for lo in (head * d, (h + g) * d, (h + kv + g) * d)]
            o, lse = _exact_head(c, *leaves, 0, c["causal"], n if c["train"] and n <= 8192 else 4096)
            out["o"][i, head], out["lse"][i, head] = o.detach(), lse.detach()
            if c["train"]:
                grads = torch.autograd.grad(o, leaves, p["dout"][i, head].double())
                out["dq"][i, head] = grads[0]
                out["dk"][i, g] += grads[1]
                out["dv"][i, g] += grads[2]
    return out


def _exact_cache(c, p):
    """The pages as (sequence, position) fill them, one sequence at a time."""
    for i, (m, n) in enumerate(zip(*_lengths(c))):
        where = torch.arange(n, device="cuda")
        yield m, n, p["table"][i].long()[where // c["page"]], where % c["page"]


def exact(case, seed):
    c, p = case, _params(case, seed)
    if c["kind"] == "rope":
        out = {"y": _turned(c, p["x"], p["positions"])}
        if c["train"]:
            out["dx"] = _turned(c, p["dy"], -p["positions"])
        return out
    if c["kind"] == "packed":
        if work(c)["flops"] > 5e12:
            return None
        return _exact_packed(c, p)
    if c["kind"] == "append":
        k_pages, v_pages, at = p["k_pages"].double(), p["v_pages"].double(), 0
        for m, n, page, row in _exact_cache(c, p):
            new = p["kv"][at:at + m]
            k_pages[page[n - m:], :, row[n - m:]] = _turned(c, new[:, 0], torch.arange(n - m, n, device="cuda"))
            v_pages[page[n - m:], :, row[n - m:]] = new[:, 1].double()
            at += m
        return {"k_pages": k_pages, "v_pages": v_pages}
    o, at = torch.empty(p["q"].shape, dtype=torch.float64, device="cuda"), 0
    for m, n, page, row in _exact_cache(c, p):
        k, v = (p[t][page, :, row].double() for t in ("k_pages", "v_pages"))
        for head in range(c["heads"]):
            g = head * c["kv_heads"] // c["heads"]
            q = p["q"][at:at + m, head].double()
            o[at:at + m, head] = _exact_head(c, q, k[:, g], v[:, g], n - m, True, 1024)[0]
        at += m
    return {"o": o}
