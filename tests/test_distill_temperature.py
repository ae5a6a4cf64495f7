"""Temperatures that the distillation cannot use are refused, without a GPU."""
import ctypes

import pytest

import phoenix_core_b200 as pcb
from phoenix_core_b200 import _lib


@pytest.fixture(scope="module")
def library():
    from phoenix_core_b200.csrc import build
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("temperature,taken", [(1e-45, False), (1e-39, False), (2.9e-39, False), (3.5e-39, False), (4.2e-39, False), (4.3e-39, True), (1e-30, True), (0.1, True), (1e9, True), (1.8e19, True), (1.9e19, False), (3e38, False)])
def test_reciprocal_and_square(library, temperature, taken):
    """Both are taken in fp32: log2(e) / T multiplies the logits, T^2 the second term. (A call without samples is checked and does nothing.)"""
    d = _lib.DistillDesc()
    d.dtype, d.algebra, d.batch, d.units, d.entries, d.alpha, d.temperature = _lib.PCB_F16, 0, 0, 250, 4, 0.5, temperature
    status = library.pcb_distill_fwd(ctypes.byref(d), None, None, None, None, None, None, None)
    assert status == (_lib.PCB_OK if taken else _lib.PCB_ERR_INVALID_ARGUMENT)
    if taken:
        pcb.DistillDescriptor((8, 250), 4, 0.5, temperature)
    else:
        assert b"temperature" in library.pcb_last_error_message()
        with pytest.raises(ValueError, match="temperature"):
            pcb.DistillDescriptor((8, 250), 4, 0.5, temperature)
