"""The embedding, affine layer norm and linear cross entropy as ops of lazy
streams: their values and gradients, alone and as a language model's training
step, against 64 bits on the CPU.

Tolerances of a step: every product sums at most 512 terms in f32, off by at
most 512 * 2^-24 = 3e-5 of the terms' magnitudes; a gradient passes through
about ten products and as many row operations one after another, so its norm
is off by at most 20 * 3e-5 = 6e-4 of itself where the terms do not cancel.
Single ops are held to the bounds of operators_ref.py."""
import numpy as np
import pytest
import torch

import operators_ref as R
from oxidizedmlx_amd import abi, nn, synth
from oxidizedmlx_amd import backend as hb
from oxidizedmlx_amd.opkind import NodeInput, OpKind, meta
from oxidizedmlx_amd.tensor import Tensor, eval_all, value_and_grad

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]

F32, EPS = abi.F32, 1e-5


@pytest.fixture(params=[False, True], ids=["sync", "async"])
def stream(request):
    s = hb.HipStream(async_eval=request.param)
    yield s
    s.close()


def const(a, s):
    return Tensor.from_f32_on_stream(a, np.shape(a), s)


def grads_of(y, dy, wrt, s):
    """Gradients of sum(y dy)."""
    _, g = value_and_grad(y.mul(const(dy, s)).sum_all(), wrt)
    eval_all([y, *g])
    return [t.to_numpy().astype(np.float64) for t in (y, *g)]


@pytest.mark.parametrize("shape", [(6, 33), (4, 7, 64), (130,)])
def test_layer_norm_affine(stream, shape):
    cols = shape[-1]
    x, dy = synth.normal(1, shape, 0.5, 2.0), synth.normal(2, shape)
    w, b = synth.normal(3, (cols,), 1.0, 0.2), synth.normal(4, (cols,))
    t = [const(a, stream) for a in (x, w, b)]
    y, dx, dw, db = grads_of(nn.LayerNorm(cols, EPS, t[1], t[2])(t[0]), dy, t, stream)
    x2, dy2 = x.reshape(-1, cols), dy.reshape(-1, cols)
    R.check(y.reshape(-1, cols), *R.layer_norm(x2, w, b, EPS, F32), "y")
    for got, (v, bound) in zip((dx.reshape(-1, cols), dw, db), R.layer_norm_vjp(dy2, x2, w, EPS, F32)):
        R.check(got, v, bound, "gradient")


@pytest.mark.parametrize("scale", [None, 1.0, 8.0])
def test_embedding(stream, scale):
    vocab, dim = 57, 24
    ids = (synth.uniform01(5, 60) ** 2 * (vocab + 4)).astype(np.int32) - 2   # some out of range
    w, dy = synth.normal(1, (vocab, dim)), synth.normal(2, (5, 12, dim))
    W = const(w, stream)
    y, dw = grads_of(nn.Embedding(W, scale)(const(ids.reshape(5, 12).astype(np.float32), stream)), dy, [W], stream)
    s = 1.0 if scale is None else scale
    R.check(y.reshape(60, dim), *R.embedding(w, ids, s, F32), "y")
    R.check(dw, *R.embedding_vjp(dy.reshape(60, dim), ids, vocab, s, F32), "dw")


@pytest.mark.parametrize("frozen", ["", "x", "w"])
def test_linear_cross_entropy(stream, frozen):
    rows, dim, vocab = 70, 48, 333
    x, w = synth.normal(1, (rows, dim)), synth.normal(2, (vocab, dim), 0.0, 0.3)
    t = (synth.uniform01(3, rows) * vocab).astype(np.float32)
    t = np.floor(t)
    t[::5], t[1::9], t[2::11], t[3::13] = -100, np.nan, vocab, np.inf
    g = synth.normal(4, (rows,))
    X, W = const(x, stream), const(w, stream)
    wrt = [a for a, n in ((X, "x"), (W, "w")) if n != frozen]
    got = grads_of(X.linear_cross_entropy(W, const(t, stream)), g, wrt, stream)
    ids = np.where((t >= 0) & (t < vocab), np.nan_to_num(t, posinf=0), -1).astype(np.int32)
    want = R.cross_entropy(x, w, ids, F32)[:1]
    # The stream's gradient takes lse from the loss: one sum of dim terms and
    # two roundings more, under twice the bound of the logits.
    grads = [(v, 2 * b) for v, b in R.cross_entropy_vjp(x, w, ids, g, F32)]
    want += [p for p, n in zip(grads, "xw") if n != frozen]
    for a, (v, b) in zip(got, want):
        R.check(a, v, b, f"frozen {frozen!r}")


def test_eval_node_with_host_values(hip):
    b = hb.HipBackend()
    x, w, t = synth.normal(1, (9, 16)), synth.normal(2, (40, 16)), np.arange(9, dtype=np.float32)
    out = b.eval_node(OpKind.LinearCrossEntropy, [NodeInput(x, (9, 16)), NodeInput(w, (40, 16)), NodeInput(t, (9,))], meta([9]))
    R.check(out.astype(np.float64), *R.cross_entropy(x, w, t.astype(np.int32), F32)[0], "loss")
    with pytest.raises(abi.ShapeMismatch):
        b.eval_node(OpKind.LinearCrossEntropy, [NodeInput(x, (9, 16)), NodeInput(w, (16, 40)), NodeInput(t, (9,))], meta([9]))
    with pytest.raises(abi.ShapeMismatch):
        b.eval_node(OpKind.LayerNormAffine(EPS), [NodeInput(x, (9, 16)), NodeInput(t, (9,)), NodeInput(t, (9,))], meta([9, 16]))
    with pytest.raises(abi.InvalidArgument):
        b.eval_node(OpKind.ScaledEmbedding(1.0), [NodeInput(w, (40, 16))], meta([9, 16]))
    with pytest.raises(abi.ShapeMismatch):
        b.eval_node(OpKind.EmbeddingVjp(1.0), [NodeInput(x, (9, 16)), NodeInput(t, (9,))], meta([40, 17]))


def test_ids_and_targets_have_no_gradient(stream):
    w, ids = const(synth.normal(1, (7, 4)), stream), const(np.arange(3, dtype=np.float32), stream)
    with pytest.raises(abi.InvalidArgument, match="VJP not implemented"):
        value_and_grad(w.scaled_embedding(ids, 1.0).sum_all(), [ids])
    x = const(synth.normal(2, (3, 4)), stream)
    with pytest.raises(abi.InvalidArgument, match="VJP not implemented"):
        value_and_grad(x.linear_cross_entropy(w, ids).sum_all(), [ids])


def test_shapes_are_checked_when_built(stream):
    x, w = const(synth.normal(1, (3, 4)), stream), const(synth.normal(2, (7, 5)), stream)
    with pytest.raises(abi.ShapeMismatch):
        x.linear_cross_entropy(w, const(np.zeros(3, np.float32), stream))
    with pytest.raises(abi.ShapeMismatch):
        x.linear_cross_entropy(const(synth.normal(2, (7, 4)), stream), const(np.zeros(4, np.float32), stream))
    with pytest.raises(abi.ShapeMismatch):
        x.layer_norm_affine(const(np.ones(4, np.float32), stream), const(np.ones(3, np.float32), stream), EPS)
    with pytest.raises(abi.InvalidArgument):
        nn.LayerNorm(4, EPS, weight=const(np.ones(4, np.float32), stream))


# ── a language model's training step ──────────────────────────────────────

def torch_loss(cfg, p, tokens, targets):
    b, s = tokens.shape
    x = p["embedding"][torch.tensor(tokens.reshape(-1)).long()]
    rms = lambda v: v / torch.sqrt(v.square().mean(-1, keepdim=True) + cfg.eps)
    heads = lambda v: v.reshape(b, s, cfg.n_heads, -1).transpose(1, 2)
    mask = torch.full((s, s), -1e9, dtype=torch.float64).triu(1)
    for i in range(cfg.n_layers):
        w = {k.split(".")[2]: v for k, v in p.items() if k.startswith(f"layers.{i}.")}
        a = rms(x)
        q, k, v = (heads(a @ w["w" + n].T + w["b" + n]) for n in "qkv")
        att = torch.softmax(q @ k.transpose(-1, -2) / (cfg.d_model // cfg.n_heads) ** 0.5 + mask, -1) @ v
        x = x + (att.transpose(1, 2).reshape(b * s, -1) @ w["wo"].T + w["bo"])
        x = x + (torch.nn.functional.silu(rms(x) @ w["w1"].T + w["b1"]) @ w["w2"].T + w["b2"])
    z = rms(x) @ p["lm_head"].T
    return torch.nn.functional.cross_entropy(z, torch.tensor(targets.reshape(-1)).long(), ignore_index=-100)


def test_decoder_training_step(stream):
    """DecoderLM.loss: loss and every parameter's gradient (the keys' bias has
    none: it moves all of a row's scores alike)."""
    cfg = nn.DecoderConfig(n_layers=2, d_model=64, n_heads=2, vocab=517, max_batch=2, max_seq=32)
    values = nn.decoder_params(cfg, 3, std=0.1)
    rng = np.random.default_rng(4)
    tokens = rng.integers(0, cfg.vocab, (2, 24))
    targets = np.roll(tokens, -1, 1)
    targets[:, -1] = -100
    targets[0, :5] = -100
    lm = nn.DecoderLM(cfg, stream, values)
    params = {n: t for n, t in lm.parameters().items() if not n.endswith(".bk")}
    loss, grads = value_and_grad(lm.loss(tokens, targets), list(params.values()))
    eval_all([loss, *grads])
    p = {"embedding": values["embedding"], "lm_head": values["lm_head"]}
    p.update({f"layers.{i}.{n}": v for i, lp in enumerate(values["layers"]) for n, v in lp.items()})
    p = {n: torch.tensor(v, dtype=torch.float64, requires_grad=True) for n, v in p.items()}
    want = torch_loss(cfg, p, tokens, targets)
    assert abs(float(loss.to_numpy()) - want.item()) <= 6e-4 * abs(want.item())
    exact = torch.autograd.grad(want, [p[n] for n in params])
    for n, g, e in zip(params, grads, exact):
        e = e.numpy()
        off = np.linalg.norm(g.to_numpy().astype(np.float64) - e) / np.linalg.norm(e)
        print(f"{n}: {off:.2e}", flush=True)
        assert off <= 6e-4, n


def test_a_model_of_the_three_operators(stream):
    """Scaled embedding, layer norm with weight and bias, cross entropy with the
    embedding as its own output projection: the tied weight's gradient is the
    sum of both ends'."""
    vocab, dim, n = 301, 40, 90
    w = synth.normal(1, (vocab, dim), 0.0, 0.2)
    g, b = synth.normal(2, (dim,), 1.0, 0.1), synth.normal(3, (dim,), 0.0, 0.1)
    ids = (synth.uniform01(4, n) ** 3 * vocab).astype(np.int32)
    targets = np.roll(ids, -1)
    targets[-1] = -1
    W, G, B = (const(a, stream) for a in (w, g, b))
    x = nn.Embedding(W, dim ** 0.5)(const(ids.astype(np.float32), stream))
    loss, grads = value_and_grad(nn.LinearCrossEntropy(W)(nn.LayerNorm(dim, EPS, G, B)(x), targets), [W, G, B])
    eval_all([loss, *grads])
    t = [torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in (w, g, b)]
    h = torch.nn.functional.layer_norm(t[0][torch.tensor(ids).long()] * dim ** 0.5, (dim,), t[1], t[2], EPS)
    want = torch.nn.functional.cross_entropy(h @ t[0].T, torch.tensor(targets).long(), ignore_index=-1)
    assert abs(float(loss.to_numpy()) - want.item()) <= 6e-4 * want.item()
    for a, e in zip(grads, torch.autograd.grad(want, t)):
        e = e.numpy()
        assert np.linalg.norm(a.to_numpy().astype(np.float64) - e) <= 6e-4 * np.linalg.norm(e)


def test_no_row_with_a_target(stream):
    w, x = const(synth.normal(1, (11, 8)), stream), const(synth.normal(2, (5, 8)), stream)
    loss, grads = value_and_grad(nn.LinearCrossEntropy(w)(x, np.full(5, -100)), [x, w])
    eval_all([loss, *grads])
    assert float(loss.to_numpy()) == 0.0
    assert not any(g.to_numpy().any() for g in grads)


def test_steps_on_one_stream(stream):
    """Three training steps that each clear the stream: the same bits from the
    same inputs."""
    w0, x0, t = synth.normal(1, (300, 64)), synth.normal(2, (128, 64)), np.arange(128) * 2
    seen = []
    for _ in range(3):
        stream.clear()
        w, x = const(w0, stream), const(x0, stream)
        loss, grads = value_and_grad(nn.LinearCrossEntropy(w)(x, t), [x, w])
        eval_all([loss, *grads])
        seen.append([a.to_numpy() for a in (loss, *grads)])
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            np.testing.assert_array_equal(a, b)
