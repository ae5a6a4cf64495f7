"""The dense layer in 8 bits against its definition in 64 bits: every algebra, both filter layouts, the types, sizes around the blocks of
128, the tiles and the cuts of the reduction, in forward, both gradients and the filter's quantisation."""
import pytest
import torch

import dense8_reference as ref
import phoenix_core_b200 as pcb
from phoenix_core_b200.descriptors import MULTIVECTOR_DIM

pytestmark = pytest.mark.gpu

ALGEBRAS = {"real": pcb.Algebra.REAL, "complex": pcb.Algebra.COMPLEX, "quaternion": pcb.Algebra.QUATERNION, "ga300": pcb.Algebra.GA_300}
LAYOUTS = {"io": pcb.FilterLayout.IO, "oi": pcb.FilterLayout.OI}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def make(algebra, layout, dtype, n, i, o, seed=0):
    gen = torch.Generator().manual_seed(seed + 1000 * n + 10 * i + o)
    dim, t = MULTIVECTOR_DIM[ALGEBRAS[algebra]], DTYPES[dtype]

    def normal(*shape):
        return torch.randn(shape, generator=gen)

    x = (normal(dim * n, i) * normal(1, i).exp()).to(t)
    w = normal(dim, i, o) * (1.0 / (dim * i)) ** 0.5
    w = (w if layout == "io" else w.transpose(1, 2)).contiguous().to(t)
    dy = (normal(dim * n, o) * normal(1, o).exp() * 2.0 ** -6).to(t)
    bias = normal(dim, o).to(t)
    if algebra == "real":
        w, bias = w[0], bias[0]
    return dim, x, w, bias, dy


def run(algebra, layout, x, w, bias, dy, need_dx=True):
    a, l = ALGEBRAS[algebra], LAYOUTS[layout]
    xd, wd, dyd = x.cuda(), w.cuda(), dy.cuda()
    fwd = pcb.DenseFwdDescriptor(tuple(x.shape), tuple(w.shape), a, l, bias is not None)
    bwd = pcb.DenseBwdDescriptor(tuple(x.shape), tuple(w.shape), a, l, need_dx)
    f8 = pcb.Filter8(tuple(w.shape), a, l)
    pcb.quantizeFilter8(wd, f8)
    y = torch.full(fwd.getOutputShape(), float("nan"), dtype=x.dtype, device="cuda")
    pcb.dense8Fwd(xd, f8, None if bias is None else bias.cuda(), y, fwd)
    dw = torch.full(w.shape[:-2] + (bwd.getInputChannels(), bwd.getOutputChannels()), float("nan"), dtype=x.dtype, device="cuda")
    dx = torch.full(tuple(x.shape), float("nan"), dtype=x.dtype, device="cuda") if need_dx else None
    pcb.dense8Bwd(xd, f8, dyd, dw, dx, bwd)
    torch.cuda.synchronize()
    pcb.ops.Device.get(xd.device).checkStatus()
    return f8, y, dw, dx


def check(got, want, size, summed, dtype, what):
    got, want = got.double().cpu(), want.reshape(got.shape)
    bound = ref.bound(want, size.reshape(got.shape), summed, dtype)
    bad = (got - want).abs() - bound
    bad = torch.where(torch.isnan(bad), torch.full_like(bad, float("inf")), bad)
    assert (bad <= 0).all(), "%s: off by %.3e where %.3e is allowed" % (what, (got - want).abs().flatten()[bad.argmax()], bound.flatten()[bad.argmax()])


def verify(algebra, layout, dtype, n, i, o, with_bias=True):
    dim, x, w, bias, dy = make(algebra, layout, dtype, n, i, o)
    f8, y, dw, dx = run(algebra, layout, x, w, bias if with_bias else None, dy)
    t = DTYPES[dtype]
    w8 = ref.quantized(w.double().reshape(dim, *w.shape[-2:]), 128, 128)
    assert torch.equal(f8.dequantize().double().cpu().reshape(w8.shape), w8), "filter"
    w_io = w8 if layout == "io" else w8.transpose(1, 2).contiguous()
    x64, dy64 = x.double().reshape(dim, n, i), dy.double().reshape(dim, n, o)
    want, size = ref.forward(dim, x64, w_io, bias.double().reshape(dim, o) if with_bias else None)
    check(y, want, size + (bias.double().reshape(dim, 1, o).abs() if with_bias else 0.0), dim * i, t, "y")
    dx64, sx, dw64, sw = ref.backward(dim, x64, w_io, dy64)
    check(dx, dx64, sx, dim * o, t, "dx")
    check(dw, dw64, sw, dim * n, t, "dw")


# one value, one block, around a block; K cut into groups of four blocks; tokens around the narrow tiles (16, 64, 128) and above
SIZES = [(1, 1, 1), (1, 128, 128), (3, 127, 129), (16, 130, 40), (17, 520, 257), (64, 96, 512), (65, 1100, 60), (128, 384, 100), (129, 512, 136), (300, 640, 300)]


@pytest.mark.parametrize("n,i,o", SIZES)
@pytest.mark.parametrize("layout", ["io", "oi"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_real(n, i, o, layout, dtype):
    verify("real", layout, dtype, n, i, o)


@pytest.mark.parametrize("n,i,o", [(1, 33, 17), (16, 128, 128), (50, 200, 130), (130, 64, 96), (260, 250, 131)])
@pytest.mark.parametrize("layout", ["io", "oi"])
@pytest.mark.parametrize("algebra", ["complex", "quaternion", "ga300"])
def test_algebras(n, i, o, layout, algebra):
    verify(algebra, layout, "bf16" if n % 2 else "f16", n, i, o)


@pytest.mark.parametrize("layout,dtype", [("io", "bf16"), ("oi", "f16"), ("oi", "f32")])
def test_wide_tiles(layout, dtype):
    """More tiles of 256 columns than two for each SM."""
    verify("real", layout, dtype, 2309, 260, 5000, with_bias=dtype != "f16")


def test_special_values():
    """Blocks of zeros, of the smallest numbers, of one large one; infinities and NaN reach the rows that hold them and no other."""
    n, i, o = 6, 256, 130
    dim, x, w, bias, dy = make("real", "io", "f32", n, i, o)
    x[0] = 0.0
    x[1] = 2.0 ** -140
    x[2, :128] = 0.0
    x[2, 5] = 3.0e38
    w = w * 2.0 ** -20
    x[3, 7] = float("inf")
    x[4, 200] = float("nan")
    f8, y, dw, dx = run("real", "io", x, w, None, dy)
    w8 = ref.quantized(w.double()[None], 128, 128)
    x8 = ref.rows_by_128(x.double()[None])
    assert torch.equal(f8.dequantize().double().cpu()[None], w8)
    want, size = ref.product(1, x8, w8)
    got = y.double().cpu()
    for row in (0, 1, 2, 5):
        assert ((got[row] - want[0, row]).abs() <= ref.bound(want[0, row], size[0, row], i, torch.float32)).all(), row
    assert (got[0] == 0).all() and torch.isnan(got[3]).all() and torch.isnan(got[4]).all()
    bad = torch.zeros(i, dtype=torch.bool)
    bad[7] = bad[200] = True
    assert torch.equal(torch.isnan(dw).all(dim=1).cpu(), bad) and torch.equal(torch.isnan(dw).any(dim=1).cpu(), bad)
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,i,o", [(2, 1100, 300), (9, 2052, 130), (16, 3000, 64), (5, 513, 20000), (7, 1026, 19100)])
def test_few_tokens(n, i, o, dtype):
    """Tokens that the product quantises itself: long reductions cut over CTAs, features of every alignment, more tiles than SMs."""
    verify("real", "oi" if o % 4 else "io", dtype, n, i, o)


def test_few_tokens_special_values():
    n, i, o = 3, 300, 70
    dim, x, w, bias, dy = make("complex", "oi", "bf16", n, i, o)
    x[1, 200] = float("inf")
    x[0] = 0.0
    x[dim * n - 1, 3] = float("nan")
    f8, y, _, _ = run("complex", "oi", x, w, None, dy)
    y = y.reshape(dim, n, o)
    assert torch.isnan(y[:, 1]).all() and torch.isnan(y[:, 2]).all() and torch.isfinite(y[:, 0]).all()
