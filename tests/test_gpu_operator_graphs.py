"""The affine layer norm, embedding and linear cross entropy entry points in
recorded graphs: replays equal the eager results, with eager work in between,
and two graphs recorded on one stream may replay on two streams at once, as each
holds its own workspaces."""
import threading

import numpy as np
import pytest

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


class Step:
    """Embedding, layer norm and loss of one batch, forward and backward."""

    def __init__(self, seed, n, dim, vocab, dt):
        w = R.rounded(synth.normal(seed, (vocab, dim), 0.0, 1.0), dt)
        ids = (synth.uniform01(seed + 1, n) ** 3 * vocab).astype(np.int32)
        t = np.roll(ids, -1)
        t[::7] = -100
        self.n, self.dim, self.vocab, self.dt = n, dim, vocab, dt
        self.w, self.head = R.Dev(w, dt), R.Dev(R.rounded(w * 0.1, dt), dt)
        self.g, self.b = (R.Dev(R.rounded(synth.normal(seed + k, (dim,), 1.0, 0.1), dt), dt) for k in (2, 3))
        self.ids, self.t = R.Dev(ids, abi.I32), R.Dev(t, abi.I32)
        self.dloss = R.Dev(np.full(n, 1 / n, np.float32))
        self.x, self.h, self.dh, self.dx = (R.Dev(dt=dt, shape=(n, dim)) for _ in range(4))
        self.loss, self.lse = R.Dev(shape=(n,)), R.Dev(shape=(n,))
        self.dhead, self.dw = (R.Dev(dt=dt, shape=(vocab, dim)) for _ in range(2))
        self.dg, self.db = (R.Dev(dt=dt, shape=(dim,)) for _ in range(2))
        self.outs = [self.x, self.h, self.loss, self.lse, self.dh, self.dhead, self.dx, self.dg, self.db, self.dw]

    def run(self, s):
        n, d, v, dt = self.n, self.dim, self.vocab, self.dt
        hb.embedding_rows(dt, self.w.ptr, self.ids.ptr, self.x.ptr, n, v, d, 2.0, s)
        hb.layernorm_affine_rows(dt, self.x.ptr, self.g.ptr, self.b.ptr, self.h.ptr, n, d, 1e-5, s)
        hb.linear_cross_entropy(dt, self.h.ptr, self.head.ptr, self.t.ptr, self.loss.ptr, self.lse.ptr, n, d, v, s)
        hb.linear_cross_entropy_vjp(dt, self.h.ptr, self.head.ptr, self.t.ptr, self.lse.ptr, self.dloss.ptr, self.dh.ptr,
                                    self.dhead.ptr, n, d, v, s)
        hb.layernorm_affine_vjp_rows(dt, self.dh.ptr, self.x.ptr, self.g.ptr, self.dx.ptr, self.dg.ptr, self.db.ptr, n, d,
                                     1e-5, s)
        hb.embedding_vjp_rows(dt, self.dx.ptr, self.ids.ptr, self.dw.ptr, n, v, d, 2.0, s)

    def spoil(self):
        for o in self.outs:
            o.buf.upload(np.full(o.n * o.size, 0xFF, np.uint8), o.at)

    def results(self):
        return [o.get() for o in self.outs]


@pytest.fixture
def streams():
    s = [hb.create_stream() for _ in range(3)]
    yield s
    for x in s:
        hb.destroy_stream(x)


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
@pytest.mark.parametrize("n,dim,vocab", [(300, 136, 1003), (20000, 8, 300)])
def test_replays_equal_the_eager_run(streams, n, dim, vocab, dt):
    s = streams[0]
    step, other = Step(1, n, dim, vocab, dt), Step(50, 40, 72, 555, dt)
    step.run(s)
    hb.synchronize(s)
    want = step.results()
    with hb.Graph(s) as g:
        step.run(s)
    for rep in range(4):
        step.spoil()
        other.run(s)            # eager work on the recording stream between replays
        other.run(None)
        hb.synchronize()
        g.launch()
        hb.synchronize(s)
        for a, b in zip(step.results(), want):
            np.testing.assert_array_equal(a, b, err_msg=f"replay {rep}")
    g.close()


@pytest.mark.parametrize("dt", R.DTYPES, ids=R.NAMES.get)
def test_two_graphs_of_one_stream_replay_at_once(streams, dt):
    s, s1, s2 = streams
    steps = [Step(1, 1500, 264, 4001, dt), Step(2, 1500, 264, 4001, dt)]
    want, graphs = [], []
    for step in steps:
        step.run(s)
        hb.synchronize(s)
        want.append(step.results())
        with hb.Graph(s) as g:
            step.run(s)
        graphs.append(g)
    for rep in range(6):
        for step in steps:
            step.spoil()
        hb.synchronize()
        for g, on in zip(graphs, (s1, s2)):
            g.launch(on)
        steps_eager = Step(9, 700, 264, 4001, dt) if rep == 3 else None
        if steps_eager:
            steps_eager.run(s)   # and eager work on the stream they were recorded on
        hb.synchronize()
        for step, w in zip(steps, want):
            for a, b in zip(step.results(), w):
                np.testing.assert_array_equal(a, b, err_msg=f"replay {rep}")
    for g in graphs:
        g.close()


@pytest.mark.parametrize("dt", [abi.F32, abi.BF16], ids=R.NAMES.get)
def test_two_streams_at_once(streams, dt):
    steps = [Step(1, 1500, 264, 4001, dt), Step(2, 1300, 264, 4001, dt)]
    want = []
    for step in steps:
        step.run(None)
        hb.synchronize()
        want.append(step.results())
        step.spoil()
    for rep in range(4):
        for step, s in zip(steps, streams):
            step.run(s)
        hb.synchronize()
        for step, w in zip(steps, want):
            for a, b in zip(step.results(), w):
                np.testing.assert_array_equal(a, b, err_msg=f"pass {rep}")


def test_a_recording_without_memory_fails_and_leaves_the_stream_usable(streams):
    """A recorded call whose workspace cannot be allocated is an error; the
    stream then runs and records as before."""
    s = streams[0]
    L = abi.load_library()
    step = Step(1, 300, 136, 1003, abi.BF16)
    step.run(s)
    hb.synchronize(s)
    want = step.results()
    with pytest.raises(abi.FfiFailed):
        with hb.Graph(s):
            L.mlxhip_debug_fail_allocations(0)
            try:
                step.run(s)
            finally:
                L.mlxhip_debug_fail_allocations(-1)
    step.spoil()
    step.run(s)
    hb.synchronize(s)
    for a, b in zip(step.results(), want):
        np.testing.assert_array_equal(a, b)
    with hb.Graph(s) as g:
        step.run(s)
    step.spoil()
    g.launch()
    hb.synchronize(s)
    for a, b in zip(step.results(), want):
        np.testing.assert_array_equal(a, b)
    g.close()


@pytest.mark.parametrize("dt", [abi.F32, abi.BF16], ids=R.NAMES.get)
def test_threads_on_one_stream(streams, dt):
    """Calls of several threads on one stream share its workspaces, one after
    the other: the kernels of a call stay together."""
    steps = [Step(k + 1, 900 + 50 * k, 72, 1003, dt) for k in range(3)]
    want = []
    for step in steps:
        step.run(streams[0])
        hb.synchronize(streams[0])
        want.append(step.results())
    for rep in range(5):
        for step in steps:
            step.spoil()
        hb.synchronize()
        threads = [threading.Thread(target=lambda step=step: [step.run(streams[0]) for _ in range(4)]) for step in steps]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        hb.synchronize(streams[0])
        for step, w in zip(steps, want):
            for a, b in zip(step.results(), w):
                np.testing.assert_array_equal(a, b, err_msg=f"repetition {rep}")


def test_a_graph_freed_while_another_is_recorded(streams):
    """The recording goes on, and nothing of it changes with the other's workspaces."""
    s = streams[0]
    steps = [Step(k + 1, 300, 136, 1003, abi.BF16) for k in range(3)]
    want = []
    for step in steps:
        step.run(s)
        hb.synchronize(s)
        want.append(step.results())
    with hb.Graph(s) as first:
        steps[0].run(s)
    first.launch()
    hb.synchronize(s)
    with hb.Graph(s) as second:
        steps[1].run(s)
        first.close()
    with hb.Graph(s) as third:
        steps[2].run(s)
    for rep in range(3):
        for step in steps:
            step.spoil()
        steps[0].run(s)
        second.launch()
        third.launch()
        hb.synchronize(s)
        for step, w in zip(steps, want):
            for a, b in zip(step.results(), w):
                np.testing.assert_array_equal(a, b, err_msg=f"replay {rep}")
    second.close()
    third.close()
