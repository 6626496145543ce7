"""Freeing a recorded graph: it waits for its own last launch and nothing else, and
its workspaces return to the pool whatever is being recorded meanwhile."""
import threading
import time

import numpy as np
import pytest
import torch

import operators_ref as R
from oxidizedmlx_amd import abi, synth
from oxidizedmlx_amd import backend as hb
from test_gpu_lifecycle import free_device_bytes
from test_gpu_operator_graphs import Step

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("hip")]


@pytest.fixture
def streams():
    s = [hb.create_stream() for _ in range(3)]
    yield s
    for x in s:
        hb.destroy_stream(x)


class Busy:
    """A few hundred ms of products on a stream."""

    def __init__(self, stream, n=4096, times=500):
        a = hb.DeviceBuffer.from_array(synth.bf16_bits(synth.normal(1, (n, n))))
        self.held = a, hb.DeviceBuffer(4 * n * n)
        for _ in range(times):
            for _ in range(4):
                hb.gemm(abi.BF16, abi.F32, False, False, n, n, n, a, n, a, n, self.held[1], n, stream=stream)


def test_a_free_does_not_wait_for_other_streams(streams):
    step = Step(1, 300, 136, 1003, abi.BF16)
    with hb.Graph(streams[0]) as g:
        step.run(streams[0])
    g.launch()
    hb.synchronize(streams[0])
    busy = Busy(streams[1])
    t0 = time.perf_counter()
    g.close()
    t1 = time.perf_counter()
    hb.synchronize(streams[1])
    t2 = time.perf_counter()
    print(f"free {1e3 * (t1 - t0):.2f} ms, the other stream {1e3 * (t2 - t1):.2f} ms more", flush=True)
    assert t2 - t1 > t1 - t0
    del busy


def test_a_free_waits_for_its_own_launch(streams):
    """Freed at once behind a launch, its workspaces then taken by an eager call:
    both have the right results."""
    s, other = streams[:2]
    steps = [Step(k + 1, 1500, 264, 4001, abi.BF16) for k in range(2)]
    want = []
    for step in steps:
        step.run(s)
        hb.synchronize(s)
        want.append(step.results())
    for rep in range(4):
        with hb.Graph(s) as g:
            steps[0].run(s)
        for step in steps:
            step.spoil()
        hb.synchronize()
        busy = Busy(s, times=20)
        g.launch()
        g.close()
        steps[1].run(other)
        hb.synchronize()
        for step, w in zip(steps, want):
            for a, b in zip(step.results(), w):
                np.testing.assert_array_equal(a, b, err_msg=f"repetition {rep}")
        del busy


def test_a_free_waits_for_a_launch_on_the_null_stream(streams):
    steps = [Step(k + 1, 1500, 264, 4001, abi.BF16) for k in range(2)]
    want = []
    for step in steps:
        step.run(streams[0])
        hb.synchronize(streams[0])
        want.append(step.results())
    for rep in range(4):
        with hb.Graph(streams[0]) as g:
            steps[0].run(streams[0])
        for step in steps:
            step.spoil()
        hb.synchronize()
        busy = Busy(None, times=20)
        g.launch(0)
        g.close()
        steps[1].run(streams[1])
        hb.synchronize()
        for step, w in zip(steps, want):
            for a, b in zip(step.results(), w):
                np.testing.assert_array_equal(a, b, err_msg=f"repetition {rep}")
        del busy


def test_a_free_lets_other_threads_have_workspaces(streams):
    """While one thread's free waits for a long launch, another's calls go on."""
    step = Step(1, 300, 136, 1003, abi.BF16)
    other = Step(2, 300, 136, 1003, abi.BF16)
    other.run(streams[1])
    hb.synchronize()
    with hb.Graph(streams[0]) as g:
        step.run(streams[0])
    busy = Busy(streams[0])
    g.launch()
    t = threading.Thread(target=g.close)
    t.start()
    time.sleep(0.02)
    assert t.is_alive()
    other.run(streams[1])   # asks for the stream's workspaces
    assert t.is_alive()
    t.join()
    hb.synchronize()
    del busy


class Large:
    """A call with some 300 MiB of workspace."""

    def __init__(self):
        r, d, v = 8192, 64, 10000
        self.size = r, d, v
        self.x, self.w = R.Dev(R.rounded(synth.normal(1, (r, d)), abi.BF16), abi.BF16), R.Dev(np.zeros((v, d)), abi.BF16)
        self.t, self.row = R.Dev(np.arange(r, dtype=np.int32), abi.I32), R.Dev(np.ones(r, np.float32))
        self.dx, self.dw = R.Dev(dt=abi.BF16, shape=(r, d)), R.Dev(dt=abi.BF16, shape=(v, d))

    def run(self, s):
        hb.linear_cross_entropy_vjp(abi.BF16, self.x.ptr, self.w.ptr, self.t.ptr, self.row.ptr, self.row.ptr, self.dx.ptr,
                                    self.dw.ptr, *self.size, s)


def held_by(rounds):
    """Device memory that 6 calls of ``rounds`` take beyond what two do."""
    for _ in range(2):
        rounds()
    hb.synchronize()
    before = free_device_bytes()
    for _ in range(6):
        rounds()
    hb.synchronize()
    return before - free_device_bytes()


def test_graphs_freed_while_others_are_recorded_return_their_workspaces(streams):
    call, small = Large(), Step(1, 300, 136, 1003, abi.BF16)

    def rounds():
        with hb.Graph(streams[0]) as g:
            call.run(streams[0])
        g.launch()
        with hb.Graph(streams[1]) as h:
            small.run(streams[1])
            g.close()
        h.launch()
        hb.synchronize(streams[1])
        h2 = hb.Graph(streams[1])
        with h2:
            h.close()
        h2.close()

    assert held_by(rounds) < 300 << 20


def test_a_stream_destroyed_while_it_is_recorded(streams):
    """Its recording's workspaces return, and later graphs' do too."""
    call = Large()

    def rounds():
        s = hb.create_stream()
        abi.check(hb.lib().mlxhip_graph_begin(s))
        call.run(s)
        hb.destroy_stream(s)
        with hb.Graph(streams[0]) as g:
            call.run(streams[0])
        g.launch()
        g.close()

    assert held_by(rounds) < 300 << 20


def test_a_free_during_another_capture_of_the_thread(streams):
    """A graph freed while its thread captures by other means leaves that capture whole."""
    step = Step(1, 300, 136, 1003, abi.BF16)
    x, y = torch.arange(1000.0, device="cuda"), torch.zeros(1000, device="cuda")
    with hb.Graph(streams[0]) as g:
        step.run(streams[0])
    g.launch()
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        y.copy_(x * 2.0)
        g.close()
    for rep in range(3):
        x.add_(1.0)
        y.zero_()
        captured.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(y.cpu().numpy(), 2.0 * (np.arange(1000.0) + rep + 1))
