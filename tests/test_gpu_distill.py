"""Distillation from a teacher's largest logits against its definition in 64 bits: algebras, types, temperatures, vocabularies around the vectors and the
cuts of a row, rows without label or entries, masked logits, classes named twice."""
import pytest
import torch

import phoenix_core_b200 as pcb
from phoenix_core_b200.descriptors import MULTIVECTOR_DIM

pytestmark = pytest.mark.gpu

ALGEBRAS = {"real": pcb.Algebra.REAL, "complex": pcb.Algebra.COMPLEX, "quaternion": pcb.Algebra.QUATERNION, "ga300": pcb.Algebra.GA_300}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")


def make(dim, t, n, units, k, seed=0, spread=2.0):
    gen = torch.Generator().manual_seed(seed + n * 31 + units * 7 + k)
    z = (torch.randn((n, dim * units), generator=gen) * spread).to(t)
    labels = torch.randint(0, dim * units, (n,), generator=gen)
    index = torch.stack([torch.randperm(dim * units, generator=gen)[:k] for _ in range(n)]) if k else torch.zeros((n, 0), dtype=torch.int64)
    teacher = (torch.randn((n, k), generator=gen) * 2.0 + 3.0).to(t)
    grad = torch.rand((n,), generator=gen) + 0.5
    return z, labels, teacher, index, grad


def stacked(z, dim):
    n = z.shape[0]
    return z.reshape(n, dim, -1).transpose(0, 1).reshape(dim * n, -1).contiguous()


def run(dim, algebra, z, labels, teacher, index, grad, alpha, temperature):
    x = stacked(z, dim).cuda()
    d = pcb.DistillDescriptor(tuple(x.shape), index.shape[1], alpha, temperature, algebra)
    dev = lambda t: None if t is None else t.cuda()                   # noqa: E731
    loss, stats = torch.full((z.shape[0],), float("nan"), device="cuda"), torch.empty(d.getStatsShape(), device="cuda")
    dz = torch.full_like(x, float("nan"))
    args = (dev(labels), dev(teacher), dev(index))
    pcb.distillFwd(x, *args, loss, stats, d)
    pcb.distillBwd(x, *args, stats, grad.cuda(), dz, d)
    torch.cuda.synchronize()
    return loss.cpu(), dz.cpu().reshape(dim, z.shape[0], -1).transpose(0, 1).reshape(z.shape)


def reference(z, labels, teacher, index, grad, alpha, temperature):
    """Row by row from the definition. Returns loss, gradient, and the sum of the absolute terms of each."""
    z, t = z.double(), teacher.double() / temperature
    n, classes = z.shape
    loss, dz = torch.zeros(n, dtype=torch.float64), torch.zeros_like(z)
    size_l, size_g = torch.zeros(n, dtype=torch.float64), torch.zeros_like(z)
    for r in range(n):
        if (z[r] == -INF).all():
            continue
        top = z[r].max()
        if labels is not None and 0 <= labels[r] < classes and alpha < 1.0:
            q = torch.softmax(z[r], 0)
            loss[r] += (1 - alpha) * -torch.log_softmax(z[r], 0)[labels[r]]
            size_l[r] += (1 - alpha) * (1 + torch.log_softmax(z[r], 0)[labels[r]].abs() + 2 * (z[r, labels[r]] - top).abs())
            g = (1 - alpha) * q
            size_g[r] += g * (1 + (z[r] - top).abs().clamp(max=1e30))
            g[labels[r]] -= 1 - alpha
            size_g[r, labels[r]] += 1 - alpha
            dz[r] += g
        keep = [i for i in range(index.shape[1]) if 0 <= index[r, i] < classes]
        if keep and alpha > 0.0 and (t[r, keep] > -INF).any():
            logp, logq, q = torch.log_softmax(t[r, keep], 0), torch.log_softmax(z[r] / temperature, 0), torch.softmax(z[r] / temperature, 0)
            g = alpha * temperature * q
            size_g[r] += g * (1 + (z[r] - top).abs().clamp(max=1e30) / temperature)
            for i, lp in zip(keep, logp):
                p = lp.exp()
                if p > 0:
                    loss[r] += alpha * temperature ** 2 * p * (lp - logq[index[r, i]])
                    size_l[r] += alpha * temperature ** 2 * p * (1 + lp.abs() + logq[index[r, i]].abs() + (t[r, keep].max() - t[r, i]).abs()) * (2 + (z[r, index[r, i]] - top).abs() / temperature)
                    g[index[r, i]] -= alpha * temperature * p
                    size_g[r, index[r, i]] += alpha * temperature * p * (2 + (t[r, keep].max() - t[r, i]).abs())
            dz[r] += g
    size_g = torch.nan_to_num(size_g, nan=0.0)
    return loss, dz * grad.double()[:, None], size_l, size_g * grad.double().abs()[:, None]


def check(dim, algebra, t, z, labels, teacher, index, grad, alpha, temperature):
    loss, dz = run(dim, algebra, z, labels, teacher, index, grad, alpha, temperature)
    want, wdz, size_l, size_g = reference(z, labels, teacher, index, grad, alpha, temperature)
    # An exponential is off by four units in the last place (CUDA's bound for exp2f is two; the square of one has twice that) and by its argument's rounding, relative to the
    # argument, which the sizes hold; a row's sum of positive terms by its chain: the classes over the 128 threads at least, and 16 joints.
    # Then a handful of products and quotients, and one rounding to the type.
    chain = (64 + z.shape[1] / 128) * 2.0 ** -24
    ok = (loss.double() - want).abs() <= chain * size_l + 2.0 ** -24 * want.abs() + 1e-37
    assert (ok | (loss.double() == want)).all(), (loss.double() - want).abs().max()
    half, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    bound = chain * size_g * (1 + half) + half * wdz.abs() + tiny + 1e-37
    off = (dz.double() - wdz).abs()
    assert (off <= bound).all(), "off by %g, %g allowed" % (off.max(), bound.flatten()[(off - bound).argmax()])


@pytest.mark.parametrize("units", [1, 2, 9, 250, 1000, 4097, 33001])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 1.7])
def test_vocabularies(units, dtype, temperature):
    n, k = (5, min(units, 20))
    check(1, pcb.Algebra.REAL, DTYPES[dtype], *make(1, DTYPES[dtype], n, units, k), 0.6, temperature)


@pytest.mark.parametrize("algebra,units", [("complex", 77), ("quaternion", 250), ("quaternion", 5003), ("ga300", 16), ("ga300", 6001)])
@pytest.mark.parametrize("alpha", [0.0, 0.5, 1.0])
def test_algebras(algebra, units, alpha):
    dim = MULTIVECTOR_DIM[ALGEBRAS[algebra]]
    check(dim, ALGEBRAS[algebra], torch.float16, *make(dim, torch.float16, 7, units, 12), alpha, 2.0)


@pytest.mark.parametrize("n", [1, 3, 300, 700])
def test_rows(n):
    check(1, pcb.Algebra.REAL, torch.bfloat16, *make(1, torch.bfloat16, n, 520, 5), 0.5, 2.0)


@pytest.mark.parametrize("k", [0, 1, 64, 700])
def test_entries(k):
    check(4, pcb.Algebra.QUATERNION, torch.float32, *make(4, torch.float32, 4, 250, k), 0.5, 3.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_holes(dtype):
    """No label, no entry, fewer entries than places, classes out of range, a class named twice, masked logits, a row of nothing, logits of -infinity
    in the teacher's, and the lowest value of the type as a mask."""
    t, n, units, k = DTYPES[dtype], 12, 300, 8
    z, labels, teacher, index, grad = make(4, t, n, units, k)
    labels[0] = -100
    labels[1] = 4 * units
    index[2] = -1
    index[3, 3:] = -1
    index[4, 2] = index[4, 5]
    index[4, 1] = labels[4]
    index[5, 0] = 4 * units
    z[6] = -INF
    z[7, 100:900] = -INF
    labels[7], index[7] = 5, torch.arange(k)
    z[8] = torch.finfo(t).min
    z[9, 1:] = torch.finfo(t).min
    labels[9], index[9] = 0, -1
    teacher[10, 1:] = -INF
    teacher[11] = -INF
    for alpha in (0.0, 0.4, 1.0):
        for temperature in (1.0, 2.0):
            check(4, pcb.Algebra.QUATERNION, t, z, labels, teacher, index, grad, alpha, temperature)


def test_masked_class_that_the_teacher_wants():
    """A class with q = 0 and p > 0 makes the loss infinite, its gradient stays finite."""
    z, labels, teacher, index, grad = make(1, torch.float32, 2, 50, 3)
    z[0, index[0, 0]] = -INF
    labels[0] = (index[0, 0] + 1) % 50
    loss, dz = run(1, pcb.Algebra.REAL, z, labels, teacher, index, grad, 0.5, 2.0)
    assert loss[0] == INF and torch.isfinite(loss[1]) and torch.isfinite(dz).all()


def test_not_a_number_stays_in_its_row():
    z, labels, teacher, index, grad = make(1, torch.float32, 4, 5000, 3)
    z[1, 77] = float("nan")
    z[2] = float("nan")
    loss, dz = run(1, pcb.Algebra.REAL, z, labels, teacher, index, grad, 0.5, 2.0)
    assert torch.isnan(loss[1]) and torch.isnan(loss[2]) and torch.isfinite(loss[[0, 3]]).all()
    assert torch.isnan(dz[1]).all() and torch.isnan(dz[2]).all() and torch.isfinite(dz[[0, 3]]).all()


def test_large_logits():
    """Logits of several thousand: differences decide."""
    check(1, pcb.Algebra.REAL, torch.float32, *make(1, torch.float32, 6, 777, 9, spread=3000.0), 0.5, 2.0)


def test_gradient_against_differences():
    z, labels, teacher, index, grad = make(2, torch.float32, 6, 40, 5)
    grad = torch.ones(6)
    _, dz = run(2, pcb.Algebra.COMPLEX, z, labels, teacher, index, grad, 0.3, 2.0)
    direction = torch.randn(z.shape, generator=torch.Generator().manual_seed(1))
    step = 2.0 ** -6
    up, down = (run(2, pcb.Algebra.COMPLEX, z + s * direction, labels, teacher, index, grad, 0.3, 2.0)[0].double() for s in (step, -step))
    slope = (up - down) / (2 * step)
    assert ((slope - (dz.double() * direction.double()).sum(1)).abs() <= 2.0 ** -8 * (dz.double() * direction.double()).abs().sum(1)).all()


def test_rows_that_start_anywhere():
    """Logits and gradients as views of larger buffers, on any two places within sixteen bytes."""
    z, labels, teacher, index, grad = make(1, torch.bfloat16, 3, 1001, 4)
    want = run(1, pcb.Algebra.REAL, z, labels, teacher, index, grad, 0.5, 2.0)
    d = pcb.DistillDescriptor((3, 1001), 4, 0.5, 2.0, pcb.Algebra.REAL)
    for a, b in ((1, 1), (3, 6), (8, 5)):
        x = torch.zeros(3 * 1001 + 16, dtype=torch.bfloat16, device="cuda")[a:a + 3003].view(3, 1001)
        whole = torch.full((3 * 1001 + 16,), 7.0, dtype=torch.bfloat16, device="cuda")
        dz = whole[b:b + 3003].view(3, 1001)
        x.copy_(z)
        loss, stats = torch.empty(3, device="cuda"), torch.empty(3, 3, device="cuda")
        pcb.distillFwd(x, labels.cuda(), teacher.cuda(), index.cuda(), loss, stats, d)
        pcb.distillBwd(x, labels.cuda(), teacher.cuda(), index.cuda(), stats, grad.cuda(), dz, d)
        _, wdz, _, size = reference(z, labels, teacher, index, grad, 0.5, 2.0)
        assert ((dz.double().cpu() - wdz).abs() <= 2.0 ** -15 * size + 2.0 ** -8 * wdz.abs() + 1e-37).all()
        assert (whole[:b] == 7.0).all() and (whole[b + 3003:] == 7.0).all()
        assert torch.allclose(loss.cpu(), want[0], rtol=2.0 ** -18, atol=0)
