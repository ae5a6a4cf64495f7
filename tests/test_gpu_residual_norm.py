"""The norms of a residual block with its gate and scale against their formulas in 64 bits, and the gradients against differences: every algebra and
type, gates of every kind, widths around what a warp, a CTA's threads and the registers hold, and each part left out."""
import pytest
import torch

import phoenix_core_b200 as pcb
from phoenix_core_b200.descriptors import MULTIVECTOR_DIM

pytestmark = pytest.mark.gpu

ALGEBRAS = {"real": pcb.Algebra.REAL, "complex": pcb.Algebra.COMPLEX, "quaternion": pcb.Algebra.QUATERNION, "ga300": pcb.Algebra.GA_300}
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
ULP = 2.0 ** -24                 # half a step of fp32


class Case:
    def __init__(self, algebra, dtype, n, f, gates, scale=0.5, branch=True, pre=True, post=True, norm=True, grad_out=True, seed=0):
        self.dim, self.t, self.n, self.f, self.gates, self.scale = MULTIVECTOR_DIM[ALGEBRAS[algebra]], DTYPES[dtype], n, f, gates, scale
        gen = torch.Generator().manual_seed(seed + 7 * n + f)

        def make(rows, std=1.0, mean=0.0):
            return (torch.randn((self.dim * rows, f), generator=gen) * std + mean).to(self.t)

        self.x = make(n, 2.0)
        self.branch = make(n, 1.5) if branch else None
        self.gate = make(gates, 0.5, 1.0) if gates else None
        self.post = 1.0 + 0.3 * torch.randn(f, generator=gen) if post and branch else None
        self.pre = 1.0 + 0.3 * torch.randn(f, generator=gen) if pre and norm else None
        self.norm = norm
        self.dy = make(n, 0.1) if grad_out or not norm else None
        self.dh = make(n, 0.1) if norm else None
        self.desc = pcb.ResidualNormDescriptor((self.dim * n, f), gates, ALGEBRAS[algebra], scale, EPS)

    def rows(self, t):
        """[D * n, F] -> float64 [n, D, F]"""
        return t.double().reshape(self.dim, -1, self.f).transpose(0, 1)

    def factors(self):
        g = torch.ones(1, 1, 1, dtype=torch.float64) if self.gate is None else self.rows(self.gate).repeat_interleave(self.n // self.gates, 0)
        one = torch.ones(self.f, dtype=torch.float64)
        return g, one if self.post is None else self.post.double(), one if self.pre is None else self.pre.double()

    def forward(self):
        x, (g, post, pre) = self.rows(self.x), self.factors()
        rb = torch.zeros(self.n, 1, 1, dtype=torch.float64)
        y, size = x, x.abs()
        if self.branch is not None:
            b = self.rows(self.branch)
            rb = (b.square().mean((1, 2), keepdim=True) + EPS).rsqrt()
            add = self.scale * g * post * b * rb
            y, size = x + add, x.abs() + add.abs()
        ry = (y.square().mean((1, 2), keepdim=True) + EPS).rsqrt()
        return y, size, y * ry * pre, rb, ry

    def backward(self, y, rb, ry):
        """Gradients and the sums of the absolute values that make them."""
        g, post, pre = self.factors()
        zero = torch.zeros_like(y)
        dy = zero if self.dy is None else self.rows(self.dy)
        dx, sx, dpre, spre = dy, dy.abs(), None, None
        if self.dh is not None:
            dh, yn = self.rows(self.dh), y * ry
            t = dh * pre
            dx = dy + ry * (t - yn * (t * yn).mean((1, 2), keepdim=True))
            sx = dy.abs() + ry * (t.abs() + yn.abs() * (t * yn).abs().mean((1, 2), keepdim=True))
            dpre, spre = (dh * yn).sum((0, 1)), (dh * yn).abs().sum((0, 1))
        out = {"dx": (dx, sx), "dpre": (dpre, spre)}
        if self.branch is not None:
            u = self.rows(self.branch) * rb
            dn, sn = self.scale * g * dx, (self.scale * g).abs() * sx
            v, sv = dn * post, sn * post.abs()
            out["db"] = (rb * (v - u * (v * u).mean((1, 2), keepdim=True)), rb * (sv + u.abs() * (sv * u.abs()).mean((1, 2), keepdim=True)))
            out["dpost"] = ((dn * u).sum((0, 1)), (sn * u.abs()).sum((0, 1)))
            if self.gate is not None:
                shape = (self.gates, self.n // self.gates, self.dim, self.f)
                out["dgate"] = ((self.scale * dx * u * post).expand(self.n, self.dim, self.f).reshape(shape).sum(1),
                                (self.scale * sx * (u * post).abs()).expand(self.n, self.dim, self.f).reshape(shape).sum(1))
        return out

    def run(self):
        dev = lambda t: None if t is None else t.cuda()                              # noqa: E731
        nan = lambda t: None if t is None else torch.full_like(t, float("nan"), device="cuda")   # noqa: E731
        x, b, g, post, pre, dy, dh = (dev(t) for t in (self.x, self.branch, self.gate, self.post, self.pre, self.dy, self.dh))
        y, h, stats = nan(x) if b is not None else None, nan(x) if self.norm else None, torch.full((2, self.n), float("nan"), device="cuda")
        pcb.residualNormFwd(x, b, g, post, pre, y, h, stats, self.desc)
        dx, db, dg, dpost, dpre = nan(x), nan(b), nan(g), nan(post), nan(pre)
        pcb.residualNormBwd(y if y is not None else x, b, g, post, pre, stats, dy, dh, dx, db, dg, dpost, dpre, self.desc)
        torch.cuda.synchronize()
        return y, h, stats, {"dx": dx, "db": db, "dgate": dg, "dpost": dpost, "dpre": dpre}

    def close(self, what, got, want, allowed, t):
        got = got.double().cpu()
        if got.dim() == 2 and what not in ("stats",):
            got = self.rows(got)
        half, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
        bound = allowed + half * (want.abs() + allowed) + tiny
        off = (got - want).abs()
        assert (off <= bound).all(), "%s: off by %g, %g allowed" % (what, off.max(), bound.flatten()[(off - bound).argmax()])

    def check(self):
        """fp32 steps: a result of c roundings of terms whose absolute values add up to s is off by c * s * 2^-24. A row's sum has at most its width over
        32 threads in a chain (128 and more threads from 513 values on, 512 from 4096 on) and ten joints; a sum over samples at most their number."""
        width = self.dim * self.f
        chain = 64 + width / (32 if width <= 512 else 128 if width <= 4096 else 512)
        y, size, h, rb, ry = self.forward()
        gy, gh, stats, grads = self.run()
        # mean(y^2) is off by the errors of y, which are relative to the size of its terms
        worst = (size.square().sum((1, 2), keepdim=True) / y.square().sum((1, 2), keepdim=True).clamp(min=1e-300)).sqrt()
        allowed_y = chain * ULP * size
        if gy is not None:
            self.close("y", gy, y, allowed_y, self.t)
        if gh is not None:
            _, _, pre = self.factors()
            self.close("h", gh, h, (allowed_y * ry + 2 * chain * ULP * worst * (y * ry).abs()) * pre.abs(), self.t)
            assert ((stats[1].double().cpu() - ry.flatten()).abs() <= 2 * chain * ULP * (worst * ry).flatten()).all()
        if self.branch is not None:
            assert ((stats[0].double().cpu() - rb.flatten()).abs() <= chain * ULP * rb.flatten()).all()
        # backward from what the forward call left: y as rounded, the factors as stored
        y = self.rows(gy.cpu() if gy is not None else self.x)
        rb, ry = (stats[i].double().cpu().reshape(-1, 1, 1) for i in (0, 1))
        per_group = self.n // max(self.gates, 1)
        factor = {"dx": chain, "db": 3 * chain, "dgate": 3 * chain + per_group, "dpost": 3 * chain + self.n * self.dim, "dpre": chain + self.n * self.dim}
        for name, (want, terms) in self.backward(y, rb, ry).items():
            got = grads[name]
            assert (got is None) == (want is None or (name == "dpost" and self.post is None) or (name == "dpre" and self.pre is None)), name
            if got is not None:
                self.close(name, got, want, factor[name] * ULP * terms, torch.float32 if name in ("dpost", "dpre") else self.t)


@pytest.mark.parametrize("f", [1, 7, 8, 64, 250, 509, 512, 520, 1024, 2040, 2048, 2052, 4096, 4097, 5000, 8192])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_widths(f, dtype):
    Case("real", dtype, 37, f, 37 if f % 3 == 0 else 1).check()


@pytest.mark.parametrize("f", [8193, 16384, 16392, 20001])
def test_wide_rows(f):
    for gates in (0, 2, 6):
        Case("real", "bf16" if f % 2 else "f32", 6, f, gates).check()


@pytest.mark.parametrize("gates", [0, 1, 3, 12, 600])
@pytest.mark.parametrize("algebra,f", [("real", 512), ("complex", 129), ("quaternion", 128), ("quaternion", 509), ("ga300", 40), ("ga300", 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_and_algebras(gates, algebra, f, dtype):
    Case(algebra, dtype, 600, f, gates).check()


@pytest.mark.parametrize("n", [1, 2, 5, 130, 4099])
def test_rows(n):
    Case("quaternion", "f16", n, 96, 1).check()
    Case("real", "bf16", n, 1024, n).check()


@pytest.mark.parametrize("parts", [dict(branch=False), dict(norm=False), dict(post=False), dict(pre=False), dict(grad_out=False), dict(branch=False, pre=False, grad_out=False)])
@pytest.mark.parametrize("f", [256, 333, 9000])
def test_parts_left_out(parts, f):
    Case("complex" if f < 9000 else "real", "bf16", 50, f, 0 if parts.get("branch") is False else 5, **parts).check()


def test_more_than_thirty_two_bits_of_bytes():
    """1.1 billion values: byte offsets beyond 2^31. Rows at both ends against the formula."""
    n, f = 270000, 4096
    x = torch.randn((64, f), device="cuda").to(torch.bfloat16).repeat(n // 64 + 1, 1)[:n].contiguous()
    y, h = torch.empty_like(x), torch.empty_like(x)
    pcb.residualNormFwd(x, x, None, None, None, y, h, None, pcb.ResidualNormDescriptor((n, f)))
    for r in (0, n - 1):
        v = x[r].double()
        want = v + v * (v.square().mean() + 1e-6).rsqrt()
        assert ((y[r].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -15) * want.abs()).all()


def test_zero_rows_and_special_values():
    """A row of zeros gives zeros (epsilon), infinities and NaN stay in their rows."""
    d = pcb.ResidualNormDescriptor((4, 256))
    x, b = torch.zeros((4, 256), device="cuda"), torch.zeros((4, 256), device="cuda")
    x[1] = 1.0
    x[2, 3] = float("nan")
    b[3, 5] = float("inf")
    y, h = torch.empty_like(x), torch.empty_like(x)
    pcb.residualNormFwd(x, b, None, None, None, y, h, None, d)
    assert (y[0] == 0).all() and (h[0] == 0).all() and torch.equal(y[1], x[1]) and torch.isfinite(h[1]).all()
    assert torch.isnan(h[2]).all() and torch.isnan(h[3]).any()


def test_gradients_against_differences():
    """Directional derivatives of sum(y * a + h * c) by the calls themselves, in fp32: central differences of step e have an error of e^2 and one of the losses'
    roundings over e, both far below the 2^-7 asked for."""
    case = Case("quaternion", "f32", 12, 40, 3)
    gy, _, stats, grads = case.run()
    gen = torch.Generator().manual_seed(5)
    inputs = {"dx": case.x, "db": case.branch, "dgate": case.gate, "dpost": case.post, "dpre": case.pre}

    def loss(values):
        y, h, s = (torch.empty_like(case.x, device="cuda") for _ in range(3))
        pcb.residualNormFwd(values["dx"].cuda(), values["db"].cuda(), values["dgate"].cuda(), values["dpost"].cuda(), values["dpre"].cuda(), y, h, None, case.desc)
        return (y.double().cpu() * case.dy.double() + h.double().cpu() * case.dh.double()).sum()

    for name, value in inputs.items():
        direction = torch.randn(value.shape, generator=gen)
        step = 2.0 ** -8
        up, down = (loss({**inputs, name: value + s * direction}) for s in (step, -step))
        slope, grad = (up - down) / (2 * step), (grads[name].double().cpu() * direction.double()).sum()
        scale = (grads[name].double().cpu().abs() * direction.double().abs()).sum()
        assert (slope - grad).abs() <= 2.0 ** -7 * scale, name
