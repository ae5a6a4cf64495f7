"""The operators of a dense residual block used together: norm, 8-bit dense layers, the norms and the gate behind the block, the classifier and its
distillation loss, forward and backward. Each stage is held to its definition at the values that really reach it, autograd to the entry points, a captured
and replayed step to the eager one, calls on two streams to calls one by one; and the harness's training step with a teacher."""
import pytest
import torch

import dense8_reference as ref
import phoenix_core_b200 as pcb
from phoenix_core_b200.autograd import DistillFunction, QDense8, QDense8Function, QResidualNorm, ResidualNormFunction

pytestmark = pytest.mark.gpu

Q, IO = pcb.Algebra.QUATERNION, pcb.FilterLayout.IO
N, F, WIDE, UNITS, K = 60, 96, 200, 75, 9            # samples, features, hidden features, classes / 4, the teacher's entries


class Problem:
    def __init__(self, seed, n=N, dtype=torch.bfloat16):
        gen = torch.Generator().manual_seed(seed)

        def normal(*shape, std=1.0):
            return (torch.randn(shape, generator=gen) * std).cuda()

        self.x = normal(4 * n, F, std=2.0).to(dtype)
        self.gate = (1.0 + normal(4 * 3, F, std=0.3)).to(dtype)
        self.w = [normal(4, i, o, std=(1.0 / (4 * i)) ** 0.5).to(dtype) for i, o in ((F, WIDE), (WIDE, F), (F, UNITS))]
        self.bias = normal(4, WIDE, std=0.1).to(dtype)
        self.norm_in, self.post, self.pre = (1.0 + normal(F, std=0.1) for _ in range(3))
        self.labels = torch.randint(0, 4 * UNITS, (n,), generator=gen).cuda()
        self.index = torch.stack([torch.randperm(4 * UNITS, generator=gen)[:K] for _ in range(n)]).cuda()
        self.teacher = normal(n, K, std=2.0).to(dtype)
        self.leaves = [self.x, self.gate, *self.w, self.bias, self.norm_in, self.post, self.pre]

    def copy_(self, other):
        for a, b in zip(self.leaves + [self.labels, self.index, self.teacher], other.leaves + [other.labels, other.index, other.teacher]):
            a.copy_(b)


def autograd_step(p):
    """Losses and gradients of the leaves through torch."""
    leaves = [t.detach().requires_grad_(True) for t in p.leaves]
    x, gate, w1, w2, w3, bias, norm_in, post, pre = leaves
    y0, h0 = ResidualNormFunction.apply(x, None, None, None, norm_in, Q)
    hidden = torch.relu(QDense8Function.apply(h0, w1, bias, Q))
    branch = QDense8Function.apply(hidden, w2, None, Q)
    _, h = ResidualNormFunction.apply(y0, branch, gate, post, pre, Q, 0.5)
    logits = QDense8Function.apply(h, w3, None, Q)
    losses = DistillFunction.apply(logits, p.labels, p.teacher, p.index, 0.6, 2.0, Q)
    return [losses.detach(), *torch.autograd.grad(losses.sum(), leaves)]


def explicit_step(p):
    """The same by the entry points, with everything in between."""
    n = p.x.shape[0] // 4

    def dense(x, w, bias):
        fwd, bwd = pcb.DenseFwdDescriptor(tuple(x.shape), tuple(w.shape), Q, IO, bias is not None), pcb.DenseBwdDescriptor(tuple(x.shape), tuple(w.shape), Q, IO, True)
        f8 = pcb.Filter8(tuple(w.shape), Q, IO)
        pcb.quantizeFilter8(w, f8)
        y = torch.empty(fwd.getOutputShape(), dtype=x.dtype, device="cuda")
        pcb.dense8Fwd(x, f8, bias, y, fwd)

        def back(dy):
            dw, dx = torch.empty_like(w), torch.empty_like(x)
            pcb.dense8Bwd(x, f8, dy, dw, dx, bwd)
            return dw, dx
        return y, f8, back

    first, last = pcb.ResidualNormDescriptor(tuple(p.x.shape), 0, Q), pcb.ResidualNormDescriptor(tuple(p.x.shape), 3, Q, 0.5)
    h0, h, y = (torch.empty_like(p.x) for _ in range(3))
    s0, s1 = (torch.empty(2, n, device="cuda") for _ in range(2))
    pcb.residualNormFwd(p.x, None, None, None, p.norm_in, None, h0, s0, first)
    a, f1, back1 = dense(h0, p.w[0], p.bias)
    hidden = torch.relu(a)
    branch, f2, back2 = dense(hidden, p.w[1], None)
    pcb.residualNormFwd(p.x, branch, p.gate, p.post, p.pre, y, h, s1, last)
    logits, f3, back3 = dense(h, p.w[2], None)
    d = pcb.DistillDescriptor(tuple(logits.shape), K, 0.6, 2.0, Q)
    losses, s2, dlogits = torch.empty(n, device="cuda"), torch.empty(3, n, device="cuda"), torch.empty_like(logits)
    pcb.distillFwd(logits, p.labels, p.teacher, p.index, losses, s2, d)
    pcb.distillBwd(logits, p.labels, p.teacher, p.index, s2, torch.ones(n, device="cuda"), dlogits, d)
    dw3, dh = back3(dlogits)
    dres, dbranch, dx = (torch.empty_like(p.x) for _ in range(3))
    dgate, dpost, dpre, dnorm = torch.empty_like(p.gate), torch.empty_like(p.post), torch.empty_like(p.pre), torch.empty_like(p.norm_in)
    # y itself goes nowhere else: no gradient from the residual path behind the block
    pcb.residualNormBwd(y, branch, p.gate, p.post, p.pre, s1, None, dh, dres, dbranch, dgate, dpost, dpre, last)
    dw2, dhidden = back2(dbranch)
    da = dhidden * (a > 0)
    dw1, dh0 = back1(da)
    pcb.residualNormBwd(p.x, None, None, None, p.norm_in, s0, dres, dh0, dx, None, None, None, dnorm, first)
    dbias = da.view(4, n, -1).float().sum(1).to(da.dtype)
    between = {"h0": h0, "a": a, "hidden": hidden, "branch": branch, "y": y, "h": h, "logits": logits, "dlogits": dlogits, "dh": dh, "dbranch": dbranch, "dhidden": dhidden,
               "da": da, "dh0": dh0, "dres": dres, "f": (f1, f2, f3)}
    return [losses, dx, dgate, dw1, dw2, dw3, dbias, dnorm, dpost, dpre], between


def test_every_stage_holds_at_the_values_that_reach_it():
    p = Problem(1)
    out, b = explicit_step(p)
    half = 2.0 ** -8
    n = N

    def rows(t):
        return t.double().cpu().reshape(4, -1, t.shape[1])

    def dense_stage(x, f8, y, bias, dy, dw, dx):
        w = f8.dequantize().double().cpu()
        want, size = ref.forward(4, rows(x), w, None if bias is None else bias.double().cpu())
        assert ((rows(y) - want).abs() <= ref.bound(want, size, 4 * x.shape[1], torch.bfloat16) + (0.0 if bias is None else 2.0 ** -20)).all()
        wdx, sx, wdw, sw = ref.backward(4, rows(x), w, rows(dy))
        assert ((rows(dx) - wdx).abs() <= ref.bound(wdx, sx, 4 * y.shape[1], torch.bfloat16)).all()
        assert ((dw.double().cpu() - wdw).abs() <= ref.bound(wdw, sw, 4 * n, torch.bfloat16)).all()

    f1, f2, f3 = b["f"]
    losses, dx, dgate, dw1, dw2, dw3, dbias, dnorm, dpost, dpre = out
    dense_stage(b["h0"], f1, b["a"], p.bias, b["da"], dw1, b["dh0"])
    dense_stage(b["hidden"], f2, b["branch"], None, b["dbranch"], dw2, b["dhidden"])
    dense_stage(b["h"], f3, b["logits"], None, b["dlogits"], dw3, b["dh"])

    # the norms: forward from the formula, backward by torch in 64 bits at the same values; fp32 steps are far below the rounding to bf16 (2^-16 covers sums of 384 terms)
    def samples(t):
        return t.double().cpu().reshape(4, -1, F).transpose(0, 1)

    def norm(v, w):
        return v * (v.square().mean((1, 2), keepdim=True) + 1e-6).rsqrt() * w.double().cpu()

    def near(got, want, terms=None):
        terms = want.abs() if terms is None else terms
        assert ((samples(got) - want).abs() <= half * want.abs() + 2.0 ** -16 * (terms + want.abs().amax((1, 2), keepdim=True)) + 1e-30).all()

    near(b["h0"], norm(samples(p.x), p.norm_in))
    gate = samples(p.gate).repeat_interleave(n // 3, 0)
    y = samples(p.x) + 0.5 * gate * norm(samples(b["branch"]), p.post)
    near(b["y"], y)
    near(b["h"], norm(y, p.pre))
    leaves = [t.detach().clone().requires_grad_(True) for t in (samples(p.x), samples(b["branch"]), samples(p.gate), p.post.double().cpu(), p.pre.double().cpu())]
    x_, b_, g_, post_, pre_ = leaves
    unit = lambda v: v * (v.square().mean((1, 2), keepdim=True) + 1e-6).rsqrt()      # noqa: E731
    h_ = unit(x_ + 0.5 * g_.repeat_interleave(n // 3, 0) * unit(b_) * post_) * pre_
    grads = torch.autograd.grad((h_ * samples(b["dh"])).sum(), leaves)
    # (the call's y and dh are rounded, the formula's y is not: another half step relative to the largest of a row)
    for got, want in zip((b["dres"], b["dbranch"]), grads[:2]):
        assert ((samples(got) - want).abs() <= 3 * half * want.abs().amax((1, 2), keepdim=True)).all()
    assert ((samples(dgate) - grads[2]).abs() <= 3 * half * grads[2].abs().amax()).all()
    for got, want in ((dpost, grads[3]), (dpre, grads[4])):
        assert ((got.double().cpu() - want).abs() <= 3 * half * want.abs().amax()).all()
    z = b["logits"].double().cpu().reshape(4, n, UNITS).transpose(0, 1).reshape(n, -1).requires_grad_(True)
    prob = torch.softmax(p.teacher.double().cpu() / 2.0, 1)
    soft = (prob * (prob.log() - torch.log_softmax(z / 2.0, 1).gather(1, p.index.cpu()))).sum(1)
    want = 0.4 * torch.nn.functional.cross_entropy(z, p.labels.cpu(), reduction="none") + 0.6 * 4.0 * soft
    assert ((losses.double().cpu() - want).abs() <= 2.0 ** -18 * (1.0 + want.abs())).all()
    (dz,) = torch.autograd.grad(want.sum(), z)
    got = b["dlogits"].double().cpu().reshape(4, n, UNITS).transpose(0, 1).reshape(n, -1)
    assert ((got - dz).abs() <= half * dz.abs() + 2.0 ** -18).all()


def test_autograd_is_the_entry_points():
    p = Problem(2)
    for got, want in zip(autograd_step(p), explicit_step(p)[0]):
        assert got.dtype == want.dtype and torch.equal(got, want)


def test_the_same_call_gives_the_same_bits():
    p = Problem(3, n=300)
    first = autograd_step(p)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(autograd_step(p), first))


def test_captured_and_replayed():
    """One graph, replayed on inputs that change in place, while another stream's eager steps run in between."""
    p, others = Problem(4), [Problem(s) for s in (4, 5, 6)]
    want = [autograd_step(o) for o in others]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(2):
            autograd_step(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = autograd_step(p)
    for o, w in zip(others, want):
        p.copy_(o)
        graph.replay()
        eager = autograd_step(others[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, w))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))


def capture(p, stream):
    with torch.cuda.stream(stream):
        for _ in range(2):
            autograd_step(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = autograd_step(p)
    return graph, out


def test_two_graphs_of_one_stream_at_once():
    """Two steps captured one after the other on the same stream and replayed beside each other on two others."""
    problems = [Problem(11, n=300), Problem(12, n=300)]
    want = [autograd_step(p) for p in problems]
    stream = torch.cuda.Stream()
    graphs = [capture(p, stream) for p in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    for _ in range(20):
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_a_graph_outlives_the_workspace_of_its_stream():
    """A larger eager call on the capture's stream replaces the stream's workspace; what takes its memory is left alone by a replay."""
    p, larger = Problem(13, n=42), Problem(14, n=2001)
    want = autograd_step(p)
    stream = torch.cuda.Stream()
    graph, out = capture(p, stream)
    with torch.cuda.stream(stream):
        autograd_step(larger)
        others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert all((t == 7).all() for t in others) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    problems = [Problem(7, n=300), Problem(8, n=90)]
    want = [autograd_step(p) for p in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(5):
        for p, s, r in zip(problems, streams, results):
            with torch.cuda.stream(s):
                r.append(autograd_step(p))
    torch.cuda.synchronize()
    for r, w in zip(results, want):
        assert all(torch.equal(a, b) for step in r for a, b in zip(step, w))


def test_rows_behind_the_batch_stay():
    """Results in the front of larger buffers: nothing behind them is written."""
    n, f, o = 5, 130, 77
    x = torch.randn(4 * n, f, device="cuda").to(torch.float16)
    w = torch.randn(4, f, o, device="cuda").to(torch.float16)
    fwd, f8 = pcb.DenseFwdDescriptor((4 * n, f), (4, f, o), Q, IO, False), pcb.Filter8((4, f, o), Q, IO)
    pcb.quantizeFilter8(w, f8)
    for rows in (4 * n,):
        buffer = torch.full((rows * o + 512,), 7.0, dtype=torch.float16, device="cuda")
        pcb.dense8Fwd(x, f8, None, buffer[:rows * o].view(rows, o), fwd)
        assert (buffer[rows * o:] == 7.0).all()
    d = pcb.ResidualNormDescriptor((4 * n, f), 1, Q)
    gate = torch.ones(4, f, device="cuda", dtype=torch.float16)
    y, h = (torch.full((4 * n * f + 512,), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    stats = torch.empty(2, n, device="cuda")
    pcb.residualNormFwd(x, x, gate, None, None, y[:4 * n * f].view(4 * n, f), h[:4 * n * f].view(4 * n, f), stats, d)
    grads = [torch.full((k + 512,), 7.0, dtype=torch.float16, device="cuda") for k in (4 * n * f, 4 * n * f, 4 * f)]
    pcb.residualNormBwd(y[:4 * n * f].view(4 * n, f), x, gate, None, None, stats, x, x, grads[0][:4 * n * f].view(4 * n, f), grads[1][:4 * n * f].view(4 * n, f),
                        grads[2][:4 * f].view(4, f), None, None, d)
    for t, k in ((y, 4 * n * f), (h, 4 * n * f), (grads[0], 4 * n * f), (grads[1], 4 * n * f), (grads[2], 4 * f)):
        assert (t[k:] == 7.0).all() and not (t[:k] == 7.0).all()


def test_modules():
    torch.manual_seed(0)
    layer, norm = QDense8(F, WIDE, dtype=torch.float16), QResidualNorm(F, residual_scale=0.5)
    x = torch.randn(4 * 7, F, device="cuda").to(torch.float16)
    y = layer(x)
    y.float().square().sum().backward()
    assert layer.weight.grad.shape == layer.weight.shape and layer.bias.grad.shape == layer.bias.shape and torch.isfinite(layer.weight.grad).all()
    layer.pack()
    with torch.no_grad():
        assert torch.equal(layer(x), y)
        layer.weight.mul_(2.0)
        assert torch.equal(layer(x), y)                        # as packed
        layer.pack()
        assert not torch.equal(layer(x), y)
    real = QDense8(F, 40, algebra=pcb.Algebra.REAL, dtype=torch.bfloat16)
    z = real(torch.randn(3, F, device="cuda").to(torch.bfloat16))
    z.sum().backward()
    assert z.shape == (3, 40) and real.weight.grad.shape == (F, 40) and real.bias.grad.shape == (40,)
    first, h = norm(x)
    assert torch.equal(first, x)
    second, h2 = norm(x, h, torch.ones(4, F, device="cuda", dtype=torch.float16))
    (second.float().sum() + h2.float().square().sum()).backward()
    assert torch.isfinite(norm.post_weight.grad).all() and torch.isfinite(norm.pre_weight.grad).all()


def test_only_one_of_the_outputs_used():
    x = torch.randn(4 * 6, F, device="cuda").requires_grad_(True)
    b = torch.randn(4 * 6, F, device="cuda").requires_grad_(True)
    y, h = ResidualNormFunction.apply(x, b, None, None, None, Q)
    gx, gb = torch.autograd.grad(y.sum(), (x, b), retain_graph=True)
    assert torch.equal(gx, torch.ones_like(x)) and torch.isfinite(gb).all()
    gx, _ = torch.autograd.grad(h.sum(), (x, b))
    assert torch.isfinite(gx).all()


def test_training_step_with_a_teacher():
    """The harness's step: its loss from its own logits, a captured step equal to the eager one to within the atomically summed batch-norm statistics."""
    from phoenix_core_b200 import qresnet
    torch.backends.cudnn.enabled = False
    dev = torch.device("cuda", 0)
    g = torch.Generator(device="cpu").manual_seed(5)
    images = torch.randn((8, 3, 64, 64), generator=g).to(torch.float16).to(dev)
    labels = torch.randint(0, 1000, (8,), generator=g).to(dev)
    teacher = qresnet.Teacher((torch.randn((8, 16), generator=g) + 5.0).to(torch.float16).to(dev), torch.stack([torch.randperm(1000, generator=g)[:16] for _ in range(8)]).to(dev))
    model = qresnet.QResNet18(dev, seed=3)
    for _ in range(3):
        model.train_step(images, labels, 1, lr=0.01, teacher=teacher)
    state = [t.clone() for t in (model.flat_w32, model.flat_mom, model.bn_w, model.bn_m)]

    def restore():
        for t, v in zip((model.flat_w32, model.flat_mom, model.bn_w, model.bn_m), state):
            t.copy_(v)

    model.flat_w16.copy_(model.flat_w32)
    with torch.no_grad():
        logits = model.forward(images).double()
    eager = float(model.train_step(images, labels, 1, lr=0.01, teacher=teacher))
    prob = torch.softmax(teacher.logits.double() / 2.0, 1)
    soft = (prob * (prob.log() - torch.log_softmax(logits / 2.0, 1).gather(1, teacher.indices))).sum(1)
    want = float((0.5 * torch.nn.functional.cross_entropy(logits, labels, reduction="none") + 0.5 * 4.0 * soft).mean())
    assert abs(eager - want) <= 2e-2 * abs(want)
    restore()
    assert model.capture(images, labels, lr=0.01, teacher=teacher)
    restore()
    graphed = float(model.step(images, labels, 1, lr=0.01, teacher=teacher))
    assert abs(graphed - eager) <= 2e-2 * abs(eager) and float(model.flat_g16.float().abs().max()) > 0
    with pytest.raises(ValueError):
        model.step(images, labels, 1, lr=0.01)
