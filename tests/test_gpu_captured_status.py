"""Waits that run out in calls that a graph replays are reported as those of eager calls are. The expiry is made by the self-test's kernel, which waits a few
thousand clocks on a barrier that nothing signals and returns."""
import time

import pytest
import torch

import phoenix_core_b200 as pcb
from phoenix_core_b200 import _lib
from phoenix_core_b200.ops import _raw_stream
from test_gpu_captures import Layer, device

pytestmark = pytest.mark.gpu


def expire(dev):
    """A call whose wait runs out, issued as the operators issue theirs."""
    with dev.accessControl:
        ws = dev.requestWorkspace(4096)
        _lib.check(_lib.lib().pcb_selftest_wait_expiry(None, None, None, None, ws.data_ptr(), ws.numel(), 1 << 12, _raw_stream(dev.index)))


def reported(dev):
    try:
        dev.checkStatus()
    except _lib.BackendError as err:
        assert err.status == _lib.PCB_ERR_DEVICE_TIMEOUT and "wait expired" in str(err)
        return True
    return False


def capture(calls, stream=None):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    return graph


@pytest.fixture
def dev():
    d = device()
    reported(d)                                                    # (whatever an earlier test left)
    assert not reported(d)
    yield d
    reported(d)


def test_captured_and_replayed(dev):
    """Also where other calls of the graph, which reset what they report into, and other tensors follow the call in question."""
    layer = Layer(40)

    def calls():
        layer.run()
        expire(dev)
        layer.run()
        torch.ones(1 << 20, device="cuda").mul_(2.0)

    graph = capture(calls)
    assert not reported(dev)                                       # nothing has run yet
    for _ in range(2):
        graph.replay()
        assert reported(dev)
        assert not reported(dev)                                   # once for each replay
    clean = capture(layer.run)
    clean.replay()
    assert not reported(dev)
    layer.run()
    assert not reported(dev)


def test_replayed_on_another_stream_than_captured(dev):
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = capture(lambda: expire(dev), stream)
    with torch.cuda.stream(other):
        graph.replay()
        assert reported(dev)
        graph.replay()
    other.synchronize()
    assert reported(dev)


def test_each_graph_for_itself(dev):
    """A graph that runs clean does not hide what another reported, nor do eager calls."""
    layer, stream = Layer(40), torch.cuda.Stream()
    bad, good = capture(lambda: expire(dev), stream), capture(layer.run, stream)
    bad.replay()
    good.replay()
    with torch.cuda.stream(stream):
        layer.run()
    torch.cuda.synchronize()
    assert reported(dev)
    good.replay()
    assert not reported(dev)


def test_a_graph_that_is_gone(dev):
    """What its last replay reported is not lost with it, and what took its place starts clean."""
    graph = capture(lambda: expire(dev))
    graph.replay()
    torch.cuda.synchronize()
    graph.reset()
    del graph
    time.sleep(0.1)
    layer = Layer(40)
    clean = capture(layer.run)
    clean.replay()
    assert reported(dev)
    for _ in range(70):                                            # (the words of graphs that are gone serve again)
        clean = capture(layer.run)
        clean.replay()
        assert not reported(dev)


def test_a_kept_input(dev):
    """The workspace that a convolution's forward call keeps, captured: its word is looked at too."""
    keep = pcb.KeptInput()
    layer = Layer(40)

    def calls():
        pcb.conv2DFwd(layer.image, layer.kernel, None, layer.out[5], layer.conv, keep=keep)
        _lib.check(_lib.lib().pcb_selftest_wait_expiry(None, None, None, None, keep.workspace.data_ptr(), keep.workspace.numel(), 1 << 12, _raw_stream(dev.index)))

    graph = capture(calls)
    graph.replay()
    assert reported(dev)


def test_eager_calls_still_report(dev):
    expire(dev)
    assert reported(dev) and reported(dev)                         # until the stream's next call
    Layer(40).run()
    assert not reported(dev)


def test_checks_after_each_operation(dev):
    """With them on (PCB_CHECK_DEVICE_STATUS=1) a capture goes through as without, and what its replays report is seen by the next eager operation."""
    layer, stream = Layer(40), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer.run()
    want = layer.results()
    dev.check_after_each_op = True
    try:
        clean, bad = capture(layer.run, stream), capture(lambda: (layer.run(), expire(dev)), stream)
        clean.replay()
        assert layer.same(layer.results(), want)
        layer.run()
        bad.replay()
        with pytest.raises(_lib.BackendError, match="wait expired"):
            layer.run()
        layer.run()
    finally:
        dev.check_after_each_op = False
