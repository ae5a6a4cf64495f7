"""The backward norms leave the SMs of a margin free, as the forward norms and the products do: the grids that a capture records, and the results."""
import pytest
import torch

import phoenix_core_b200 as pcb
from test_gpu_residual_norm import Case

pytestmark = pytest.mark.gpu

# rows in registers (aligned; odd, with a CTA for each place that rows start at; gates shared by groups, and one for each value), and rows wider than those
CASES = [("real", "bf16", 2000, 1024, 0), ("quaternion", "f16", 1501, 509, 1), ("real", "f32", 1200, 515, 3), ("real", "bf16", 900, 512, 900), ("real", "f16", 700, 8200, 7)]


@pytest.fixture
def margin(request):
    before = pcb.getSmMargin()
    yield
    pcb.setSmMargin(before)


@pytest.mark.parametrize("sms", [0, 5, 64])
@pytest.mark.parametrize("algebra,dtype,n,f,gates", CASES)
def test_results(algebra, dtype, n, f, gates, sms, margin):
    pcb.setSmMargin(sms)
    Case(algebra, dtype, n, f, gates).check()


@pytest.mark.parametrize("algebra,dtype,n,f,gates", CASES)
def test_a_call_that_was_made_before_the_margin(algebra, dtype, n, f, gates, margin):
    """What a descriptor keeps (the workspace's size) suits every margin; the sums lie where they lay."""
    case = Case(algebra, dtype, n, f, gates)
    pcb.setSmMargin(0)
    case.check()
    pcb.setSmMargin(64)
    case.check()
    pcb.setSmMargin(0)
    case.check()


@pytest.mark.parametrize("sms", [0, 5, 64])
@pytest.mark.parametrize("algebra,dtype,n,f,gates", CASES)
def test_grids(algebra, dtype, n, f, gates, sms, margin):
    runtime, driver = pytest.importorskip("cuda.bindings.runtime"), pytest.importorskip("cuda.bindings.driver")

    def ok(result):
        assert int(result[0]) == 0, result[0]
        return result[1] if len(result) == 2 else result[1:]

    case = Case(algebra, dtype, n, f, gates)
    case.run()
    dev = lambda t: None if t is None else t.cuda()                                      # noqa: E731
    y, b, g, post, pre, dy, dh = (dev(t) for t in (case.x, case.branch, case.gate, case.post, case.pre, case.dy, case.dh))
    stats, empty = torch.ones((2, n), device="cuda"), lambda t: None if t is None else torch.empty_like(t)      # noqa: E731
    out = [empty(t) for t in (y, b, g, post, pre)]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    pcb.setSmMargin(sms)
    with torch.cuda.stream(stream):
        ok(runtime.cudaStreamBeginCapture(stream.cuda_stream, runtime.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed))
        try:
            pcb.residualNormBwd(y, b, g, post, pre, stats, dy, dh, *out, case.desc)
        finally:
            (graph,) = runtime.cudaStreamEndCapture(stream.cuda_stream)[1:]
    _, count = ok(driver.cuGraphGetNodes(int(graph), 0))
    nodes, _ = ok(driver.cuGraphGetNodes(int(graph), count))
    kernels = [ok(driver.cuGraphKernelNodeGetParams(node)) for node in nodes]
    ok(runtime.cudaGraphDestroy(graph))
    total = torch.cuda.get_device_properties(0).multi_processor_count
    wide = f > 8192
    main = [k for k in kernels if k.blockDimX == 512] if wide else [k for k in kernels if k.sharedMemBytes > 64 * 1024]
    assert main, [(k.gridDimX, k.blockDimX, k.sharedMemBytes) for k in kernels]
    first = main[0]
    assert first.gridDimX <= (total - sms) * (4 if wide else 1), (first.gridDimX, first.blockDimX)
