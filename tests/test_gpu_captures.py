"""What captured calls use lives as long as the graph that runs them, however the capture was begun, and no longer."""
import gc
import time

import pytest
import torch

import phoenix_core_b200 as pcb
from phoenix_core_b200.ops import Device

pytestmark = pytest.mark.gpu

Q, IO = pcb.Algebra.QUATERNION, pcb.FilterLayout.IO


def device():
    return Device.get(torch.device("cuda", torch.cuda.current_device()))


class Layer:
    """Calls that need a workspace: an 8-bit dense layer in both directions, a norm's backward call, a convolution in both directions with its kept input."""

    def __init__(self, n, seed=0, i=200, o=136):
        gen = torch.Generator().manual_seed(seed)

        def normal(*shape, std=1.0):
            return (torch.randn(shape, generator=gen) * std).cuda().half()

        self.x, self.w, self.dy = normal(4 * n, i), normal(4, i, o, std=0.04), normal(4 * n, o)
        self.f8 = pcb.Filter8(tuple(self.w.shape), Q, IO)
        pcb.quantizeFilter8(self.w, self.f8)
        self.fwd = pcb.DenseFwdDescriptor(tuple(self.x.shape), tuple(self.w.shape), Q, IO, False)
        self.bwd = pcb.DenseBwdDescriptor(tuple(self.x.shape), tuple(self.w.shape), Q, IO, True)
        self.norm = pcb.ResidualNormDescriptor(tuple(self.x.shape), 0, Q)
        self.pre = torch.ones(i, device="cuda")
        self.stats = torch.empty(self.norm.getStatsShape(), device="cuda")
        h = torch.empty_like(self.x)
        pcb.residualNormFwd(self.x, None, None, None, self.pre, None, h, self.stats, self.norm)
        self.image, self.kernel, self.dimage = normal(4 * 3, 16, 24, 24), normal(4, 16, 16, 3, 3, std=0.05), normal(4 * 3, 16, 24, 24)
        shapes = (tuple(self.image.shape), tuple(self.kernel.shape))
        self.conv = pcb.Conv2DFwdDescriptor(*shapes, (1, 1), (1, 1), pcb.Padding.SAME, (), 1, Q, pcb.DataFormat.NCHW, pcb.FilterLayout.OIHW, False, False)
        self.conv_bwd = pcb.Conv2DBwdDescriptor(*shapes, (1, 1), (1, 1), pcb.Padding.SAME, (), 1, Q, pcb.DataFormat.NCHW, pcb.FilterLayout.OIHW, True, False)
        e = torch.empty_like
        self.out = [torch.empty((4 * n, o), device="cuda", dtype=torch.half), e(self.w), e(self.x), e(self.x), e(self.pre), e(self.image), e(self.kernel), e(self.image)]

    def run(self):
        y, dw, dx, norm_dx, dpre, image, dkernel, dimage = self.out
        pcb.dense8Fwd(self.x, self.f8, None, y, self.fwd)
        pcb.dense8Bwd(self.x, self.f8, self.dy, dw, dx, self.bwd)
        pcb.residualNormBwd(self.x, None, None, None, self.pre, self.stats, None, self.x, norm_dx, None, None, None, dpre, self.norm)
        keep = pcb.KeptInput()
        pcb.conv2DFwd(self.image, self.kernel, None, image, self.conv, keep=keep)
        pcb.conv2DBwd(self.image, self.kernel, self.dimage, dkernel, dimage, self.conv_bwd, kept=keep)

    def results(self):
        torch.cuda.synchronize()
        out = [t.clone() for t in self.out]
        for t in self.out:
            t.fill_(float("nan"))
        return out


    def order(self):
        """How far two runs of the convolution's filter gradient may lie apart before they are rounded: its partial sums are added by atomics, up to three rounds of one for
        each SM, in fp32 and any order, so within 2 * 444 * 2^-24 of the sum of the absolute products (by Cauchy and Schwarz no larger than the product of the
        channels' norms)."""
        image, dimage = (t.double().transpose(0, 1).flatten(1).norm(dim=1) for t in (self.image, self.dimage))
        return 2 * 444 * 2.0 ** -24 * (dimage[:, None] * image[None, :])[None, :, :, None, None]

    def same(self, got, want):
        """Bit for bit but for the convolution's filter gradient, of which two runs lie within `order` and, rounded to fp16 each, a step (2^-10) of the value."""
        a, b = got[6].double(), want[6].double()
        return all(torch.equal(a, b) for a, b in zip(got[:6] + got[7:], want[:6] + want[7:])) and bool(((a - b).abs() <= self.order() + 2.0 ** -10 * b.abs()).all())


def take_what_is_free():
    """Tensors of every size that a call may have used, as another part of a program would make them."""
    return [torch.full((size,), 7, dtype=torch.uint8, device="cuda") for size in (1 << 10, 1 << 16, 1 << 20, 3 << 20, 1 << 23, 1 << 24) for _ in range(6)]


def test_a_capture_that_torch_does_not_know_of():
    """Begun on the stream itself: there is no memory pool of a graph behind it, and the calls' workspaces stay theirs all the same."""
    runtime = pytest.importorskip("cuda.bindings.runtime")

    def ok(result):
        assert int(result[0]) == 0, result[0]
        return result[1] if len(result) > 1 else None

    layer, stream = Layer(300), torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer.run()
        want = layer.results()
        ok(runtime.cudaStreamBeginCapture(stream.cuda_stream, runtime.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed))
        try:
            layer.run()
        finally:
            graph = ok(runtime.cudaStreamEndCapture(stream.cuda_stream))
        held = [c for c in device().captures.values() if stream.cuda_stream in c.workspaces]
        assert len(held) == 1 and held[0].others                                # the kept input of the convolution, or a workspace outgrown
        executable = ok(runtime.cudaGraphInstantiate(graph, 0))
        ok(runtime.cudaGraphDestroy(graph))
        gc.collect()
        mine = take_what_is_free()
        torch.cuda.synchronize()
        for _ in range(3):
            ok(runtime.cudaGraphLaunch(executable, stream.cuda_stream))
            assert layer.same(layer.results(), want)
            assert all((t == 7).all() for t in mine)
        ok(runtime.cudaGraphExecDestroy(executable))


def test_what_a_graph_holds_goes_with_it():
    layer, dev, stream = Layer(40), device(), torch.cuda.Stream()

    def capture():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run()
        return graph

    with torch.cuda.stream(stream):
        layer.run()
    want = layer.results()
    first = capture()
    number = max(dev.captures)
    second = capture()
    later = max(dev.captures)
    assert number in dev.captures and later > number                            # (the first lives)
    first.replay()
    assert layer.same(layer.results(), want)
    first.reset()
    del first
    for _ in range(50):                                                         # (the runtime says so on a thread of its own)
        gc.collect()
        torch.cuda.synchronize()
        time.sleep(0.02)
        third = capture()
        if number not in dev.captures:
            break
    assert number not in dev.captures
    second.reset()
    for _ in range(50):
        time.sleep(0.02)
        layer.run()                                                             # eager calls look too
        if later not in dev.captures:
            break
    assert later not in dev.captures
    second = capture()
    for graph in (second, third):
        graph.replay()
        assert layer.same(layer.results(), want)


def test_streams_of_one_capture_share_nothing():
    """Calls on two branches of one graph, which run beside each other."""
    layers, dev = [Layer(300, seed=1), Layer(310, seed=2)], device()
    wants = []
    for layer in layers:
        layer.run()
        wants.append(layer.results())
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        layers[0].run()
        with torch.cuda.stream(side):
            layers[1].run()
        main.wait_stream(side)
    c = dev.captures[max(dev.captures)]
    assert set(c.workspaces) == {main.cuda_stream, side.cuda_stream}
    for _ in range(10):
        graph.replay()
        for layer, want in zip(layers, wants):
            assert layer.same(layer.results(), want)


def test_a_kept_input_outlives_its_owner():
    """A backward call captured by itself reads what an eager forward call kept, and goes on doing so when the owner of that is gone."""
    layer, dev, stream = Layer(40), device(), torch.cuda.Stream()
    image, dkernel, dimage = layer.out[5:]
    keep = pcb.KeptInput()
    pcb.conv2DFwd(layer.image, layer.kernel, None, image, layer.conv, keep=keep)
    pcb.conv2DBwd(layer.image, layer.kernel, layer.dimage, dkernel, dimage, layer.conv_bwd, kept=keep)
    want = layer.results()
    size, order = keep.workspace.numel(), layer.order()
    pcb.conv2DFwd(layer.image, layer.kernel, None, image, layer.conv, keep=keep)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        pcb.conv2DBwd(layer.image, layer.kernel, layer.dimage, dkernel, dimage, layer.conv_bwd, kept=keep)
    assert any(t is keep.workspace for t in dev.captures[max(dev.captures)].others)
    del keep
    gc.collect()
    mine = [torch.full((size,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
    layer.image.zero_()                                                         # (the filter gradient is of what was kept)
    graph.replay()
    got = layer.results()
    assert all((t == 7).all() for t in mine) and torch.equal(got[7], want[7])
    assert ((got[6].double() - want[6].double()).abs() <= order + 2.0 ** -10 * want[6].double().abs()).all()
