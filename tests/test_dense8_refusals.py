"""What the 8-bit dense layer refuses, and the sizes that it asks for, without a GPU."""
import ctypes

import pytest
import torch

import phoenix_core_b200 as pcb
from phoenix_core_b200 import _lib

A, L = pcb.Algebra, pcb.FilterLayout


@pytest.fixture(scope="module")
def library():
    from phoenix_core_b200.csrc import build
    build.build()
    return _lib.lib()


def desc(batch=4, i=200, o=130, algebra=0, oi=0, dtype=_lib.PCB_F16, engine=_lib.ENGINE_AUTO):
    d = _lib.DenseDesc()
    d.dtype, d.batch, d.in_features, d.out_features, d.filter_oi, d.engine, d.algebra = dtype, batch, i, o, oi, engine, algebra
    return d


def test_filter8_shapes():
    f = pcb.Filter8((4, 200, 130), A.QUATERNION, L.IO, "cpu")
    assert f.values.shape == (4, 200, 130) and f.values.stride() == (200 * 144, 144, 1) and f.scales.shape == (4, 2, 2)
    f = pcb.Filter8((200, 130), A.REAL, L.OI, "cpu")
    assert f.values.shape == (200, 130) and f.scales.shape == (1, 2, 2)
    assert torch.equal(f.dequantize(), torch.zeros(200, 130))
    f.values.copy_(torch.full((200, 130), 3.0).to(torch.float8_e4m3fn))
    f.scales[0, 1, 1] = 128
    assert f.dequantize()[199, 129] == 6.0 and f.dequantize()[199, 0] == 3.0


@pytest.mark.parametrize("shape,algebra,layout", [((3, 8, 8), A.QUATERNION, L.IO), ((8, 8), A.COMPLEX, L.IO), ((4, 8, 8), A.QUATERNION, L.OIHW),
                                                  ((0, 8), A.REAL, L.IO), ((8,), A.REAL, L.IO)])
def test_filter8_refuses(shape, algebra, layout):
    with pytest.raises(ValueError):
        pcb.Filter8(shape, algebra, layout, "cpu")


def test_sizes(library):
    d = desc()
    assert library.pcb_filter8_values_size(ctypes.byref(d)) == 4 * 200 * 144
    assert library.pcb_filter8_values_size(ctypes.byref(desc(oi=1))) == 4 * 130 * 208
    assert library.pcb_filter8_scales_size(ctypes.byref(d)) == 4 * 2 * 2
    assert library.pcb_qdense8_fwd_workspace_size(ctypes.byref(d)) >= 256 + 4 * 4 * 208 + 4 * 4 * 4
    assert library.pcb_qdense8_fwd_workspace_size(ctypes.byref(desc(i=0))) == 0


def test_entry_points_refuse(library):
    d, p = desc(), 1 << 20                                     # (never read: every call below is refused before a launch)
    ws = library.pcb_qdense8_bwd_workspace_size(ctypes.byref(d)) + library.pcb_qdense8_fwd_workspace_size(ctypes.byref(d))
    fwd = library.pcb_qdense8_fwd
    assert fwd(ctypes.byref(d), None, p, p, None, p, p, ws, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert fwd(ctypes.byref(d), p, p, p, None, p, p, 16, None) == _lib.PCB_ERR_WORKSPACE
    assert fwd(ctypes.byref(d), p, p, p, None, p, None, ws, None) == _lib.PCB_ERR_WORKSPACE
    assert fwd(ctypes.byref(d), p, p, p, None, p, p + 8, ws, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert fwd(ctypes.byref(d), p, p + 8, p, None, p, p, ws, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert fwd(ctypes.byref(desc(engine=_lib.ENGINE_SIMT)), p, p, p, None, p, p, ws, None) == _lib.PCB_ERR_UNSUPPORTED
    assert fwd(ctypes.byref(desc(dtype=7)), p, p, p, None, p, p, ws, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert fwd(ctypes.byref(desc(batch=1 << 24, i=1 << 10)), p, p, p, None, p, p, 1 << 60, None) == _lib.PCB_ERR_TOO_LARGE
    assert fwd(ctypes.byref(desc(batch=0)), None, None, None, None, None, None, 0, None) == _lib.PCB_OK
    bwd = library.pcb_qdense8_bwd
    need = desc()
    need.require_input_grad = 1
    assert bwd(ctypes.byref(need), p, None, None, p, p, p, p, ws, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert bwd(ctypes.byref(need), p, p, p, p, p, None, p, ws, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert bwd(ctypes.byref(need), p, p, p, p, None, p, p, ws, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert library.pcb_quantize_filter8(ctypes.byref(d), p, p + 4, p, None) == _lib.PCB_ERR_INVALID_ARGUMENT
    assert library.pcb_quantize_filter8(ctypes.byref(d), p, p, None, None) == _lib.PCB_ERR_INVALID_ARGUMENT


def test_python_refuses():
    f = pcb.Filter8((4, 8, 16), A.QUATERNION, L.IO, "cpu")
    d = pcb.DenseFwdDescriptor((8, 8), (4, 8, 16), A.QUATERNION, L.IO, False)
    with pytest.raises(ValueError):
        pcb.quantizeFilter8(torch.zeros(4, 8, 16), f)                        # no CPU form
    with pytest.raises(ValueError):
        pcb.quantizeFilter8(torch.zeros(4, 8, 15), f)
