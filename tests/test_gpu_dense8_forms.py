"""The forms of the 8-bit product that small layers do not take, against the definition in 64 bits: pairs of SMs with tiles of 256 x 256, up to four tokens that the product
quantises itself, both gradients in one launch. The library says which form a layer takes (pcb_qdense8_form_for); each test asserts it."""
import pytest
import torch

import dense8_blocks as blocks
import dense8_reference as ref
import phoenix_core_b200 as pcb
from dense8_sizes import BOTH, FEW_TOKENS, MARGINS, PAIRS, form
from test_gpu_dense8 import DTYPES, check, make, run

pytestmark = pytest.mark.gpu


def verify(case, with_bias):
    algebra, layout, dtype, n, i, o = case
    dim, x, w, bias, dy = make(algebra, layout, dtype, n, i, o)
    f8, y, dw, dx = run(algebra, layout, x, w, bias if with_bias else None, dy)
    t = DTYPES[dtype]
    wide = lambda v, rows, cols: v.cuda().double().reshape(dim, rows, cols)               # noqa: E731
    w8 = blocks.quantized(w.cuda().double().reshape(dim, *w.shape[-2:]), 128, 128)
    assert torch.equal(f8.dequantize().double().reshape(w8.shape), w8), "filter"
    w_io = w8 if layout == "io" else w8.transpose(1, 2).contiguous()
    x64, dy64, b64 = wide(x, n, i), wide(dy, n, o), bias.cuda().double().reshape(dim, 1, o)
    want, size = blocks.forward(dim, x64, w_io)
    check(y, (want + b64 if with_bias else want).cpu(), (size + b64.abs() if with_bias else size).cpu(), dim * i, t, "y")
    dx64, sx, dw64, sw = blocks.backward(dim, x64, w_io, dy64)
    check(dx, dx64.cpu(), sx.cpu(), dim * o, t, "dx")
    check(dw, dw64.cpu(), sw.cpu(), dim * n, t, "dw")


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("case", PAIRS)
def test_pairs(case, with_bias):
    assert [form(case, p) for p in (0, 1, 2)] == [4, 4, 4]
    verify(case, with_bias)


@pytest.mark.parametrize("margin,case", MARGINS)
def test_pairs_beside_a_margin(margin, case):
    before = pcb.getSmMargin()
    pcb.setSmMargin(margin)
    try:
        assert [form(case, p) for p in (0, 1, 2)] == [4, 4, 4]
        verify(case, True)
    finally:
        pcb.setSmMargin(before)


@pytest.mark.parametrize("case", FEW_TOKENS)
def test_few_tokens(case):
    assert form(case, 0) == 1
    verify(case, True)


@pytest.mark.parametrize("case", BOTH)
def test_both_gradients(case):
    assert [form(case, p) for p in (1, 2)] == [5, 5]
    verify(case, False)


@pytest.mark.parametrize("case", [PAIRS[4], PAIRS[8]])
def test_special_values_on_pairs(case):
    """Rows of zeros and of the smallest numbers; infinities and NaN reach the rows that hold them, and in the filter gradient the features, and no other."""
    algebra, layout, dtype, n, i, o = case
    dim, x, w, _, dy = make(algebra, layout, dtype, n, i, o)
    rows = x.view(dim, n, i)
    rows[:, 0] = 0.0
    rows[:, 1] = 2.0 ** -120
    rows[0, 300, 7], rows[dim - 1, n - 1, i - 1], rows[0, 5, 130] = float("inf"), float("nan"), float("-inf")
    f8, y, dw, dx = run(algebra, layout, x, w, None, dy)
    y, dw = y.view(dim, n, o), dw.reshape(dim, i, o)
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[300, n - 1, 5]] = True
    assert torch.equal(torch.isnan(y).all(2).all(0).cpu(), bad) and torch.equal(torch.isnan(y).any(2).any(0).cpu(), bad)
    features = torch.zeros(i, dtype=torch.bool)
    features[[7, i - 1, 130]] = True
    assert torch.equal(torch.isnan(dw).all(2).all(0).cpu(), features) and torch.equal(torch.isnan(dw).any(2).any(0).cpu(), features)
    assert torch.isfinite(dx).all() and (y[:, 0] == 0).all()


@pytest.mark.parametrize("case", [PAIRS[3], PAIRS[7], FEW_TOKENS[3], FEW_TOKENS[7], BOTH[0]])
def test_the_same_bits_again(case):
    algebra, layout, dtype, n, i, o = case
    _, x, w, bias, dy = make(algebra, layout, dtype, n, i, o)
    first = run(algebra, layout, x, w, bias, dy)[1:]
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(algebra, layout, x, w, bias, dy)[1:], first))


@pytest.mark.parametrize("case", [PAIRS[7], PAIRS[2], BOTH[0], ("quaternion", "oi", "f32", 130, 200, 200), ("real", "io", "bf16", 40, 260, 260), ("complex", "io", "f16", 3, 130, 130)])
def test_the_input_gradient_in_place(case):
    """dx may replace x or, where it has its shape, dy: both are read before anything is written."""
    algebra, layout, dtype, n, i, o = case
    _, x, w, _, dy = make(algebra, layout, dtype, n, i, o)
    f8, _, dw, dx = run(algebra, layout, x, w, None, dy)
    bwd = pcb.DenseBwdDescriptor(tuple(x.shape), tuple(w.shape), f8.algebra, f8.filterLayout, True)
    places = ["x", "dy"] if i == o else ["x"]
    for place in places:
        xd, dyd, again = x.cuda(), dy.cuda(), torch.full_like(dw, float("nan"))
        target = xd if place == "x" else dyd
        pcb.dense8Bwd(xd, f8, dyd, again, target, bwd)
        assert torch.equal(again, dw) and torch.equal(target, dx), place
