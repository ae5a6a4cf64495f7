"""What the backward norms ask for, without a GPU: sums over samples, and nothing for gradients that are no sums."""
import ctypes

import pytest

from phoenix_core_b200 import _lib


@pytest.fixture(scope="module")
def library():
    from phoenix_core_b200.csrc import build
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("batch,features,algebra", [(16384, 4096, 1), (4096, 1000, 0), (512, 8200, 1), (100, 12000, 2)])
@pytest.mark.parametrize("dtype", [_lib.PCB_F32, _lib.PCB_F16])
def test_a_gate_for_each_value(library, batch, features, algebra, dtype):
    """Its gradient is written where it is made: the call needs no more than one without a gate, but for the widest cut of the sums over samples (four CTAs on each SM)."""
    d = _lib.NormDesc()
    d.dtype, d.algebra, d.batch, d.features, d.residual_scale, d.epsilon = dtype, algebra, batch, features, 1.0, 1e-6
    d.gate_rows = batch
    width = {0: 4, 1: 1, 2: 2}[algebra] * features
    assert 256 < library.pcb_residual_norm_bwd_workspace_size(ctypes.byref(d)) <= 256 + 4 * 148 * 2 * width * 4
