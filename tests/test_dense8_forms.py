"""Which form of the 8-bit product a call takes (pcb_qdense8_form_for), without a GPU: the sizes at which test_gpu_dense8_forms.py means one of them take it on a device of
148 SMs; and its reference against the one with loops."""
import ctypes

import pytest
import torch

import dense8_blocks
import dense8_reference as ref
import phoenix_core_b200 as pcb
from dense8_sizes import BOTH, FEW_TOKENS, MARGINS, PAIRS, form, sizes_of
from phoenix_core_b200 import _lib


@pytest.fixture(scope="module")
def library():
    from phoenix_core_b200.csrc import build
    build.build()
    return _lib.lib()


def test_forms(library):
    for case in PAIRS:
        assert [form(case, p) for p in (0, 1, 2)] == [4, 4, 4], case
    for case in FEW_TOKENS:
        assert form(case, 0) == 1, case
    for case in BOTH:
        assert [form(case, p) for p in (1, 2)] == [5, 5], case
    before = pcb.getSmMargin()
    try:
        for margin, case in MARGINS:
            pcb.setSmMargin(margin)
            assert [form(case, p) for p in (0, 1, 2)] == [4, 4, 4], (margin, case)
    finally:
        pcb.setSmMargin(before)
    assert form(("real", "io", "f16", 5, 4096, 4096), 0) == 2 and form(("real", "io", "f16", 64, 64, 64), 1) == 2
    assert form(("real", "io", "f16", 64, 64, 64), 2) == 3 and form(("real", "io", "f16", 4, 64, 64), 1) == 2


def test_refusals(library):
    bad = _lib.PCB_ERR_INVALID_ARGUMENT
    d = sizes_of(("real", "io", "f16", 100, 64, 64))
    assert library.pcb_qdense8_form_for(ctypes.byref(d), 3) == bad and library.pcb_qdense8_form_for(ctypes.byref(d), -1) == bad
    d.require_input_grad = 0
    assert library.pcb_qdense8_form_for(ctypes.byref(d), 1) == bad and library.pcb_qdense8_form_for(ctypes.byref(d), 2) == 3
    d.batch = 0
    assert library.pcb_qdense8_form_for(ctypes.byref(d), 0) == bad
    d.batch, d.engine = 4, _lib.ENGINE_SIMT
    assert library.pcb_qdense8_form_for(ctypes.byref(d), 0) == _lib.PCB_ERR_UNSUPPORTED


@pytest.mark.parametrize("d,r,c", [(1, 1, 1), (2, 5, 300), (1, 130, 129), (4, 200, 17)])
def test_reference(d, r, c):
    x = torch.randn((d, r, c), generator=torch.Generator().manual_seed(r), dtype=torch.float64) * 2.0 ** torch.randint(-150, 100, (d, r, 1), generator=torch.Generator().manual_seed(c))
    x[0, 0] = 0.0
    x[-1, -1, -1] = float("inf")
    same = lambda a, b: ((a == b) | (torch.isnan(a) & torch.isnan(b))).all()      # noqa: E731
    assert same(dense8_blocks.by_rows(x), ref.rows_by_128(x)) and same(dense8_blocks.by_cols(x), ref.cols_by_128(x))
    assert same(dense8_blocks.quantized(x, 128, 128), ref.quantized(x, 128, 128))
    for edge in (448.0, 448.0000001, 447.9, 3.5, 3.5000001, 2.0 ** -140):          # around the scale's steps
        x = torch.full((1, 1, 128), edge, dtype=torch.float64)
        assert same(dense8_blocks.by_rows(x), ref.rows_by_128(x))
