"""The workspace of the norms' backward call is laid out and looked after as every other call's is: a status word at its head, and no record of a staged
input survives it."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_kept_input import SHAPES, _setup

pytestmark = pytest.mark.gpu


def norm_backward(_lib, L, ws, features=256, n=2400):
    """Gradients of weights and of a gate of two rows, with the sums in `ws`."""
    d = _lib.NormDesc()
    d.dtype, d.algebra, d.batch, d.features, d.gate_rows, d.residual_scale, d.epsilon = _lib.PCB_F16, 1, n, features, 2, 1.0, 1e-6
    t = [torch.randn((n, features), device="cuda").half() for _ in range(4)]
    gate, weights = torch.randn((2, features), device="cuda").half(), [torch.ones(features, device="cuda") for _ in range(2)]
    stats = torch.ones((2, n), device="cuda")
    out = [torch.empty_like(t[0]), torch.empty_like(t[0]), torch.empty_like(gate), torch.empty_like(weights[0]), torch.empty_like(weights[0])]
    y, branch, dy, dh = t
    need = L.pcb_residual_norm_bwd_workspace_size(ctypes.byref(d))
    assert ws.numel() >= need
    _lib.check(L.pcb_residual_norm_bwd(ctypes.byref(d), y.data_ptr(), branch.data_ptr(), gate.data_ptr(), weights[0].data_ptr(), weights[1].data_ptr(), stats.data_ptr(),
                                       dy.data_ptr(), dh.data_ptr(), *(o.data_ptr() for o in out), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    return need


@pytest.fixture(scope="module")
def gpu():
    import gpu_util
    return gpu_util


def test_status_word(gpu):
    """After the call the workspace's word reads as after any call that went well, whatever the memory held before."""
    from phoenix_core_b200 import _lib
    L, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for n in (2400, 2):                                    # (sums of many parts, and groups of one row)
        ws = torch.full((1 << 24,), 0xff, dtype=torch.uint8, device="cuda")
        need = norm_backward(_lib, L, ws, n=n)
        assert L.pcb_check_device_status(ws.data_ptr(), ws.numel(), stream) == _lib.PCB_OK
        assert (ws[need:] == 0xff).all() and (ws[4:256] == 0xff).all()
    ws = torch.full((1 << 24,), 0xff, dtype=torch.uint8, device="cuda")
    norm_backward(_lib, L, ws, features=8200, n=6)         # rows wider than the registers
    assert L.pcb_check_device_status(ws.data_ptr(), ws.numel(), stream) == _lib.PCB_OK


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[3]])
def test_a_staged_input_is_forgotten(gpu, shape):
    """A convolution's forward call leaves its staged input in a workspace that the norms' backward call is given next: the convolution's filter gradient
    stages the input again."""
    from phoenix_core_b200 import _lib, ops
    x, w, dy, fwd, bwd, t, pcb = _setup(gpu, shape, "f16")
    ctx, L, stream = gpu.context("16p"), _lib.lib(), torch.cuda.current_stream().cuda_stream
    pcb.conv2DBwd(t["x"], t["w"], t["dy"], t["dw"], t["dx"], bwd, ctx)
    want = gpu.host(t["dw"])
    df = ops._conv_desc(fwd, t["x"].dtype, ctx, _lib.ENGINE_AUTO)
    db = ops._conv_desc(bwd, t["x"].dtype, ctx, _lib.ENGINE_AUTO, require_input_grad=True)
    kept = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    own = torch.empty(L.pcb_qconv2d_bwd_workspace_size(ctypes.byref(db)), dtype=torch.uint8, device="cuda")
    p = {k: v.data_ptr() for k, v in t.items()}
    _lib.check(L.pcb_qconv2d_fwd(ctypes.byref(df), p["x"], p["w"], None, p["y"], kept.data_ptr(), kept.numel(), stream))
    norm_backward(_lib, L, kept)
    t["dw"].fill_(float("nan"))
    _lib.check(L.pcb_qconv2d_bwd_kept(ctypes.byref(db), p["x"], p["w"], p["dy"], p["dw"], p["dx"], kept.data_ptr(), kept.numel(), own.data_ptr(), own.numel(), stream))
    # the same kernel on the same staged values; only the order of the atomic additions may differ (as where kept and plain backward passes are compared)
    got = gpu.host(t["dw"])
    assert np.abs(got - want).max() <= 1e-3 * np.abs(want).max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("algebra,n,f", [("real", 40, 8200), ("real", 1300, 8193), ("quaternion", 9, 2100), ("complex", 7, 5001)])
def test_gates_of_wide_rows(algebra, n, f, dtype):
    """A gate for each value, and shared ones, of rows wider than the registers."""
    from test_gpu_residual_norm import Case
    for gates in (n, 1):
        Case(algebra, dtype, n, f, gates).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_that_start_anywhere(dtype):
    """The same of tensors that do not start on 16 bytes, which take the same kernel whatever their width."""
    import phoenix_core_b200 as pcb
    from test_gpu_block_edges import guarded, shifted
    from test_gpu_residual_norm import Case
    case = Case("real", dtype, 300, 130, 300)
    y, _, stats, want = case.run()
    b, g, post, pre, dy, dh = (t.cuda() for t in (case.branch, case.gate, case.post, case.pre, case.dy, case.dh))
    out = {k: shifted(want[k], 1, float("nan")) for k in ("dx", "db", "dgate", "dpost", "dpre")}
    pcb.residualNormBwd(y, b, g, post, pre, stats, dy, dh, *(out[k][1] for k in ("dx", "db", "dgate", "dpost", "dpre")), case.desc)
    torch.cuda.synchronize()
    width = case.f
    for k, (whole, got) in out.items():
        assert guarded(whole, 1, got.numel()), k
        # each side is within its own bound of the definition (Case.check): chains of 64 + width / 32 steps of 2^-24, three of them, of terms that are no larger than
        # eight times the largest result here, and one rounding each
        step = torch.finfo(got.dtype).eps
        count = case.n if k in ("dpost", "dpre") else 0
        assert ((got.double() - want[k].double()).abs() <= step * want[k].double().abs() + 2 * (3 * (64 + width / 32) + count) * 2.0 ** -24 * 8 * want[k].double().abs().max()).all(), k
