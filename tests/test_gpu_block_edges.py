"""Calls of the block operators at the edges of what they accept: tensors that start anywhere, no samples, gates of a few odd rows, copies of layers
that have run, losses of one term where the other is infinite, logits of more than 2^31 values."""
import copy
import pickle

import pytest
import torch

import dense8_reference as ref
import phoenix_core_b200 as pcb
from phoenix_core_b200.autograd import DistillFunction, QDense8, QDense8Function, ResidualNormFunction
from test_gpu_dense8 import check as check_dense
from test_gpu_dense8 import make as make_dense
from test_gpu_dense8 import run as run_dense
from test_gpu_distill import check as check_distill
from test_gpu_distill import make as make_distill
from test_gpu_residual_norm import DTYPES, Case

pytestmark = pytest.mark.gpu

Q, R, IO = pcb.Algebra.QUATERNION, pcb.Algebra.REAL, pcb.FilterLayout.IO
GUARD = 7.0


def shifted(t, places, fill=None):
    """A copy of a tensor that starts `places` values into its buffer, which holds GUARD around it (`fill`: in it too)."""
    whole = torch.full((t.numel() + places + 16,), GUARD, dtype=t.dtype, device="cuda")
    out = whole[places:places + t.numel()].view(t.shape)
    out.copy_(t) if fill is None else out.fill_(fill)
    return whole, out


def guarded(whole, places, count):
    return (whole[:places] == GUARD).all() and (whole[places + count:] == GUARD).all()


@pytest.mark.parametrize("gates", [100, 120, 200, 300])
@pytest.mark.parametrize("algebra,f", [("real", 509), ("quaternion", 129), ("real", 4098), ("ga300", 3)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_of_few_rows(gates, algebra, f, dtype):
    """Groups of two to six samples, fewer than there are places within 16 bytes for odd rows to start at, and as many."""
    Case(algebra, dtype, 600, f, gates).check()


@pytest.mark.parametrize("algebra,f", [("real", 700), ("real", 1030), ("quaternion", 375), ("real", 1537), ("complex", 1150), ("real", 2560), ("real", 2561), ("ga300", 300)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_widths_of_every_number_of_warps(algebra, f, dtype):
    for gates in (0, 4, 60):
        Case(algebra, dtype, 60, f, gates).check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,f,gates", [(9, 512, 3), (70, 130, 1), (3, 8200, 3)])
def test_norm_tensors_start_anywhere(dtype, n, f, gates):
    """Results as from tensors on 16 bytes up to the order of sums (2 * 64 + width / 32 fp32 steps of the terms, and a rounding that falls the other way), nothing around them touched."""
    case = Case("real", dtype, n, f, gates)
    y, h, stats, grads = case.run()
    for places in (1, 3):
        put = lambda t: None if t is None else shifted(t, places)                  # noqa: E731
        x, b, g, post, pre, dy, dh = (put(t)[1] for t in (case.x, case.branch, case.gate, case.post, case.pre, case.dy, case.dh))
        out = {k: shifted(t, places, float("nan")) for k, t in dict(y=y, h=h, stats=stats, **grads).items()}
        o = {k: v[1] for k, v in out.items()}
        pcb.residualNormFwd(x, b, g, post, pre, o["y"], o["h"], o["stats"], case.desc)
        o["y"].copy_(y)                                  # (the backward call's own inputs the same in both)
        o["stats"].copy_(stats)
        pcb.residualNormBwd(o["y"], b, g, post, pre, o["stats"], dy, dh, o["dx"], o["db"], o["dgate"], o["dpost"], o["dpre"], case.desc)
        torch.cuda.synchronize()
        want = dict(y=y, h=h, stats=stats, **grads)
        for k, (whole, got) in out.items():
            assert guarded(whole, places, got.numel()), k
            ours, theirs = got.double(), want[k].double()
            # sums over rows (the weights' and the gate's) have terms of either sign: their size bounds them by the largest terms
            size = theirs.abs() + (theirs.abs().max() if k in ("dx", "db", "dgate", "dpost", "dpre") else 0.0)
            step = torch.finfo(want[k].dtype).eps
            assert ((ours - theirs).abs() <= step * theirs.abs() + (128 + f / 32) * 2.0 ** -24 * size * 4 + 1e-30).all(), k


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,i,o", [(3, 256, 128), (40, 128, 136), (200, 130, 257), (300, 512, 256)])
def test_dense8_tensors_start_anywhere(dtype, n, i, o):
    """The same bits as from tensors on 16 bytes (the cut of a call depends on its sizes alone), nothing around the results touched."""
    _, x, w, bias, dy = make_dense("quaternion", "oi", dtype, n, i, o)
    f8, y, dw, dx = run_dense("quaternion", "oi", x, w, bias, dy)
    a, l = Q, pcb.FilterLayout.OI
    fwd, bwd = pcb.DenseFwdDescriptor(tuple(x.shape), tuple(w.shape), a, l, True), pcb.DenseBwdDescriptor(tuple(x.shape), tuple(w.shape), a, l, True)
    for places in (1, 5):
        again = pcb.Filter8(tuple(w.shape), a, l)
        pcb.quantizeFilter8(shifted(w, places)[1], again)
        assert torch.equal(again.dequantize(), f8.dequantize())
        xs, bs, dys = (shifted(t, places)[1] for t in (x, bias, dy))
        out = {k: shifted(t, places, float("nan")) for k, t in dict(y=y, dw=dw, dx=dx).items()}
        pcb.dense8Fwd(xs, again, bs, out["y"][1], fwd)
        pcb.dense8Bwd(xs, again, dys, out["dw"][1], out["dx"][1], bwd)
        torch.cuda.synchronize()
        for k, want in dict(y=y, dw=dw, dx=dx).items():
            assert torch.equal(out[k][1], want) and guarded(out[k][0], places, want.numel()), k


@pytest.mark.parametrize("n,i,o", [(40, 128, 136), (200, 130, 257), (600, 512, 40)])
@pytest.mark.parametrize("algebra", ["quaternion", "real"])
def test_dense8_filter_gradient_alone(algebra, n, i, o):
    """The filter's gradient without the input's is the same sum, in this call's own cut."""
    dim, x, w, _, dy = make_dense(algebra, "io", "f32", n, i, o)
    _, _, dw, dx = run_dense(algebra, "io", x, w, None, dy, need_dx=False)
    assert dx is None
    w8 = ref.quantized(w.double().reshape(dim, *w.shape[-2:]), 128, 128)
    _, _, want, size = ref.backward(dim, x.double().reshape(dim, n, i), w8, dy.double().reshape(dim, n, o))
    check_dense(dw, want, size, dim * n, torch.float32, "dw")


@pytest.mark.parametrize("margin", [2, 61, 64])
def test_dense8_beside_other_kernels(margin):
    """With SMs left free the tiles are dealt to fewer CTAs, and cut otherwise: results within the bounds of the sums."""
    dim, n, i, o = 4, 300, 200, 520
    _, x, w, bias, dy = make_dense("quaternion", "io", "f32", n, i, o)
    w8 = ref.quantized(w.double(), 128, 128)
    want, size = ref.forward(dim, x.double().reshape(dim, n, i), w8, bias.double().reshape(dim, o))
    wdx, sdx, wdw, sdw = ref.backward(dim, x.double().reshape(dim, n, i), w8, dy.double().reshape(dim, n, o))
    before = pcb.getSmMargin()
    pcb.setSmMargin(margin)
    try:
        _, y, dw, dx = run_dense("quaternion", "io", x, w, bias, dy)
    finally:
        pcb.setSmMargin(before)
    check_dense(y, want, size + bias.double().reshape(dim, 1, o).abs(), dim * i, torch.float32, "y")
    check_dense(dx, wdx, sdx, dim * o, torch.float32, "dx")
    check_dense(dw, wdw, sdw, dim * n, torch.float32, "dw")


def test_no_samples():
    """Calls without samples write no values but the zeros of the sums over samples; what does not fit is refused all the same."""
    e = lambda *s, t=torch.float16: torch.empty(s, dtype=t, device="cuda")                       # noqa: E731
    nan = lambda *s, t=torch.float16: torch.full(s, float("nan"), dtype=t, device="cuda")        # noqa: E731
    f8 = pcb.Filter8((4, 16, 24), Q, IO)
    fwd, bwd = pcb.DenseFwdDescriptor((0, 16), (4, 16, 24), Q, IO, False), pcb.DenseBwdDescriptor((0, 16), (4, 16, 24), Q, IO, True)
    pcb.dense8Fwd(e(0, 16), f8, None, e(0, 24), fwd)
    dw = nan(4, 16, 24)
    pcb.dense8Bwd(e(0, 16), f8, e(0, 24), dw, e(0, 16), bwd)
    assert (dw == 0).all()
    with pytest.raises(ValueError):
        pcb.dense8Fwd(e(0, 16), f8, None, e(0, 23), fwd)
    d = pcb.ResidualNormDescriptor((0, 16), 2, Q)
    f32, w = torch.float32, torch.ones(16, device="cuda")
    gate, dg, dpost, dpre = e(8, 16).fill_(1.0), nan(8, 16), nan(16, t=f32), nan(16, t=f32)
    pcb.residualNormFwd(e(0, 16), e(0, 16), gate, w, w, e(0, 16), e(0, 16), e(2, 0, t=f32), d)
    pcb.residualNormBwd(e(0, 16), e(0, 16), gate, w, w, e(2, 0, t=f32), e(0, 16), e(0, 16), e(0, 16), e(0, 16), dg, dpost, dpre, d)
    assert (dg == 0).all() and (dpost == 0).all() and (dpre == 0).all()
    with pytest.raises(ValueError):
        pcb.residualNormFwd(e(0, 16), e(0, 15), gate, w, w, e(0, 16), e(0, 16), None, d)
    z = pcb.DistillDescriptor((0, 250), 3, 0.5, 2.0, Q)
    i = e(0, t=torch.int64)
    pcb.distillFwd(e(0, 250), i, e(0, 3), e(0, 3, t=torch.int64), e(0, t=f32), e(3, 0, t=f32), z)
    pcb.distillBwd(e(0, 250), i, e(0, 3), e(0, 3, t=torch.int64), e(3, 0, t=f32), e(0, t=f32), e(0, 250), z)
    x, weight = torch.empty((0, 16), dtype=torch.float16, device="cuda", requires_grad=True), torch.randn((4, 16, 24), device="cuda", dtype=torch.float16, requires_grad=True)
    y, h = ResidualNormFunction.apply(x, None, None, None, w, Q)
    DistillFunction.apply(QDense8Function.apply(h, weight, None, Q), None, None, None, 0.5, 2.0, Q).sum().backward()
    assert (weight.grad == 0).all() and x.grad.shape == (0, 16)


def test_refused_by_name():
    """The operand that does not fit is named, whichever it is."""
    d = pcb.ResidualNormDescriptor((8, 16), 0, Q)
    t = lambda *s, **k: torch.zeros(s, device="cuda", **k)                                       # noqa: E731
    x, b, y, h, stats = t(8, 16), t(8, 16), t(8, 16), t(8, 16), t(2, 2)
    for wrong, name in ((dict(b=t(8, 15)), "branch"), (dict(y=t(16, 8).t()), "output"), (dict(h=t(8, 16, dtype=torch.float16)), "norm"), (dict(stats=t(2, 3)), "stats"),
                        (dict(b=b.cpu()), "branch"), (dict(h="h"), "norm"), (dict(x=t(9, 16)), "residual")):
        a = {**dict(x=x, b=b, y=y, h=h, stats=stats), **wrong}
        with pytest.raises(ValueError, match=name):
            pcb.residualNormFwd(a["x"], a["b"], None, None, None, a["y"], a["h"], a["stats"], d)
    with pytest.raises(Exception, match="shares memory"):
        pcb.residualNormFwd(x, b, None, None, None, x, h, stats, d)


def test_copies_of_what_has_run():
    layer = QDense8(48, 24, algebra=Q, dtype=torch.float16)
    x = torch.randn((4 * 5, 48), device="cuda", dtype=torch.float16)
    with torch.no_grad():
        layer.pack()
        want = layer(x)
        for again in (copy.deepcopy(layer), pickle.loads(pickle.dumps(layer))):
            assert again.filter8 is not layer.filter8 and again.filter8._storage.data_ptr() != layer.filter8._storage.data_ptr()
            assert torch.equal(again(x), want)
            again.weight.mul_(2.0)
            again.pack()
            assert not torch.equal(again(x), want) and torch.equal(layer(x), want)
    case = Case("quaternion", "f16", 6, 40, 2)
    y, h, _, grads = case.run()
    case.desc = copy.deepcopy(case.desc)
    again = case.run()
    assert torch.equal(again[1], h) and all(torch.equal(again[3][k], grads[k]) for k in grads)


def test_gradients_of_gradients_are_refused():
    """The backward calls have no derivative: asking for one is an error (torch has nothing to refuse where the gradient handed in is a constant, but no gradient to go back from either)."""
    w = torch.randn((4, 16, 24), device="cuda", requires_grad=True)
    x = torch.randn((20, 16), device="cuda", requires_grad=True)
    for loss in (QDense8Function.apply(x, w, None, Q).square().sum(), ResidualNormFunction.apply(x, x * 2.0, None, None, None, Q)[1].square().sum(),
                 DistillFunction.apply(x, torch.zeros(5, dtype=torch.int64, device="cuda"), None, None, 0.5, 1.0, Q).sum()):
        (g,) = torch.autograd.grad(loss, x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
            g.square().sum().backward()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_term_alone(dtype):
    """A masked class that the teacher wants has no say with alpha 0, a masked label none with alpha 1."""
    t = DTYPES[dtype]
    z, labels, teacher, index, grad = make_distill(4, t, 5, 300, 6)
    z[0, index[0, 2]] = -float("inf")
    z[1, labels[1]] = -float("inf")
    labels[0] = (index[0, 2] + 1) % 1200
    index[1] = torch.where(index[1] == labels[1], (index[1] + 1) % 1200, index[1])
    check_distill(4, Q, t, z[:1], labels[:1], teacher[:1], index[:1], grad[:1], 0.0, 2.0)
    check_distill(4, Q, t, z[1:2], labels[1:2], teacher[1:2], index[1:2], grad[1:2], 1.0, 2.0)


def test_more_than_thirty_two_bits_of_logits():
    """2.3 billion logits: the first and the last rows against their definition."""
    n, units = 17500, 131072
    d = pcb.DistillDescriptor((n, units), 2, 0.5, 2.0, R)
    x = torch.randn((64, units), device="cuda").to(torch.bfloat16).repeat(n // 64 + 1, 1)[:n].contiguous()
    dx = torch.empty_like(x)
    labels = torch.randint(0, units, (n,), device="cuda")
    index = torch.randint(0, units, (n, 2), device="cuda")
    teacher = torch.randn((n, 2), device="cuda").to(torch.bfloat16)
    loss, stats, grad = torch.empty(n, device="cuda"), torch.empty((3, n), device="cuda"), torch.rand(n, device="cuda") + 0.5
    pcb.distillFwd(x, labels, teacher, index, loss, stats, d)
    pcb.distillBwd(x, labels, teacher, index, stats, grad, dx, d)
    for r in (0, n // 2, n - 1):
        z = x[r].double().requires_grad_(True)
        p = torch.softmax(teacher[r].double() / 2.0, 0)
        want = -0.5 * torch.log_softmax(z, 0)[labels[r]] + 0.5 * 4.0 * (p * (p.log() - torch.log_softmax(z / 2.0, 0)[index[r]])).sum()
        (g,) = torch.autograd.grad(want, z)
        assert abs(loss[r].item() - want.item()) <= 2.0 ** -12 * abs(want.item())               # (131072 terms over 1024 threads: 2^7 steps of 2^-24, and a few more)
        off = (dx[r].double() - g * grad[r].double()).abs()
        # one rounding to bf16; fp32 steps of both sums (2^-14) of the terms, of which a class that is named has one of 0.5, 1 or 2 beside its own probability
        assert (off <= 2.0 ** -8 * g.abs() * grad[r] + 2.0 ** -14 * (g.abs() + 1e-9) * grad[r] + torch.zeros_like(off).index_fill_(0, torch.cat([labels[r:r + 1], index[r]]), 2.0 ** -13)).all()
