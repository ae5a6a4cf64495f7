"""Cases for timing the operators of a dense residual block and its training loss: the dense layer in 8-bit floating point with a
scale for each block of 128, the norms before and after a block with its gate and residual scale, and distillation from a
teacher's largest logits. Each is computed in plain torch operations or through the package's entry points.

A case is a dict of plain values; `prepare` builds what a program has in hand before the call, `run` makes one pass.

  op        "dense8", "norm" or "distill"
  mode      dense8: "fwd" (a filter kept in 8 bits) or "train" (filter quantised, forward, both gradients)
            norm: "fwd" or "bwd";  distill: "fwd" or "train" (loss and gradient)
  algebra   "real", "complex", "quaternion" or "ga300"; components are stacked on the leading axis of every tensor
  dtype     "f32", "f16" or "bf16"

The 8-bit format: a block of values is held as e4m3 numbers times 2^e, e the smallest integer with max|x| <= 448 * 2^e (0 for a
block of zeros). Activations and output gradients have blocks of 128 along the axis that the product sums over, filters blocks
of 128 x 128, each within its component.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
COMPONENTS = {"real": 1, "complex": 2, "quaternion": 4, "ga300": 8}
DEVICE = "cuda"


def _dense8(name, mode, algebra, dtype, n, ci, co, layout="oi", bias=False):
    return {"name": name, "op": "dense8", "mode": mode, "algebra": algebra, "dtype": dtype, "n": n, "ci": ci, "co": co,
            "layout": layout, "bias": bias}


def _norm(name, mode, algebra, dtype, n, features, gates, scale=1.0):
    return {"name": name, "op": "norm", "mode": mode, "algebra": algebra, "dtype": dtype, "n": n, "features": features,
            "gates": gates, "scale": scale}


def _distill(name, mode, algebra, dtype, n, units, entries, alpha, temperature, holes=False):
    return {"name": name, "op": "distill", "mode": mode, "algebra": algebra, "dtype": dtype, "n": n, "units": units,
            "entries": entries, "alpha": alpha, "temperature": temperature, "holes": holes}


def listed():
    return [
        # one token through a projection whose filter is kept in 8 bits: latency, and the filter's bytes
        _dense8("dense8_1x4096to4096_bf16_fwd", "fwd", "real", "bf16", 1, 4096, 4096, bias=True),
        # the benchmark's wide quaternion dense layer, evaluated
        _dense8("dense8_quat_256x512to512_f16_fwd", "fwd", "quaternion", "f16", 256, 512, 512, "io", True),
        # a long prompt through the widening projection of a block
        _dense8("dense8_8192x4096to8192_bf16_fwd", "fwd", "real", "bf16", 8192, 4096, 8192),
        # a square projection in training
        _dense8("dense8_8192x4096to4096_bf16_train", "train", "real", "bf16", 8192, 4096, 4096, "io"),
        # a quaternion layer in training, none of whose sizes is a round number
        _dense8("dense8_quat_777x500to1001_f16_train", "train", "quaternion", "f16", 777, 500, 1001, "io"),
        # one token between two blocks
        _norm("norm_1x4096_bf16_fwd", "fwd", "real", "bf16", 1, 4096, 1),
        # sixteen sequences of 1024 tokens between two blocks, a gate for each sequence
        _norm("norm_16384x4096_bf16_fwd", "fwd", "real", "bf16", 16384, 4096, 16, 0.5),
        # the same in the backward pass
        _norm("norm_16384x4096_bf16_bwd", "bwd", "real", "bf16", 16384, 4096, 16, 0.5),
        # a quaternion block of odd sizes with a gate for each element, backward
        _norm("norm_quat_3001x509_f16_bwd", "bwd", "quaternion", "f16", 3001, 509, 3001),
        # the classifier of the quaternion ResNet-18 (1000 classes = 250 quaternion outputs) at the harness's batch
        _distill("distill_quat_128x1000_f16_train", "train", "quaternion", "f16", 128, 250, 16, 0.5, 2.0),
        # a language model's training step: few of the teacher's logits for each of many tokens
        _distill("distill_4096x131072_bf16_train", "train", "real", "bf16", 4096, 131072, 64, 0.9, 2.0),
        # a handful of evaluated rows over an odd vocabulary, some rows without label or with part of the entries
        _distill("distill_7x50001_f32_fwd", "fwd", "real", "f32", 7, 50001, 33, 0.75, 1.5, True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


DENSE8_FLOPS = 2 * 8192 * 4096 * 4096          # a product of the listed training step
NORM_VALUES = 16384 * 4096
DISTILL_VALUES = 4096 * 131072


def draw(rng):
    """One more case of the listed ranges."""
    algebra = rng.choice(("real", "real", "complex", "quaternion", "quaternion", "ga300"))
    comps = COMPONENTS[algebra]
    dtype = rng.choice(("bf16", "f16", "f32"))
    op = rng.choice(("dense8", "dense8", "norm", "distill"))
    if op == "dense8":
        mode = rng.choice(("fwd", "train"))
        ci, co = (max(1, _log_int(rng, 64, 8192) // comps) for _ in range(2))
        room = DENSE8_FLOPS // (2 * comps * comps * ci * co)
        n = _log_int(rng, 1, max(1, min(8192, room)))
        case = _dense8(None, mode, algebra, dtype, n, ci, co, rng.choice(("io", "oi")), mode == "fwd" and rng.random() < 0.5)
    elif op == "norm":
        features = max(1, _log_int(rng, 32, 8192) // comps)
        groups = _log_int(rng, 1, 64)
        n = groups * _log_int(rng, 1, max(1, min(16384, NORM_VALUES // (comps * features)) // groups))
        case = _norm(None, rng.choice(("fwd", "bwd")), algebra, dtype, n, features, rng.choice((0, 1, groups, n)), rng.choice((1.0, 0.5, 0.1)))
    else:
        units = max(1, _log_int(rng, 16, 131072) // comps)
        bytes_left = DISTILL_VALUES * 2 // SIZES[dtype]
        n = _log_int(rng, 1, max(1, min(4096, bytes_left // (comps * units))))
        entries = min(_log_int(rng, 1, 128), comps * units)
        case = _distill(None, rng.choice(("fwd", "train")), algebra, dtype, n, units, entries, rng.choice((1.0, 0.9, 0.5)),
                        rng.choice((1.0, 1.5, 2.0, 4.0)), rng.random() < 0.5)
    del case["name"]
    return case


def work(case):
    """Bytes and operations of a pass: every input once, every output once."""
    comps, n, size = COMPONENTS[case["algebra"]], case["n"], SIZES[case["dtype"]]
    if case["op"] == "dense8":
        ci, co = case["ci"], case["co"]
        product = 2 * comps * comps * n * ci * co
        x, y, w = comps * n * ci, comps * n * co, comps * ci * co
        if case["mode"] == "fwd":
            return {"bytes": (x + y + (comps * co if case["bias"] else 0)) * size + w, "flops": product}
        return {"bytes": (2 * x + 2 * y + 2 * w) * size, "flops": 3 * product}
    if case["op"] == "norm":
        features = case["features"]
        values, gate, weights = comps * n * features, comps * case["gates"] * features, 2 * features * 4
        if case["mode"] == "fwd":
            return {"bytes": (4 * values + gate) * size + weights + 8 * n, "flops": 10 * values}
        return {"bytes": (6 * values + 2 * gate) * size + 2 * weights + 8 * n, "flops": 30 * values}
    values, pairs = comps * n * case["units"], n * case["entries"]
    teacher = pairs * (size + 8) + 8 * n
    if case["mode"] == "fwd":
        return {"bytes": values * size + teacher + 4 * n, "flops": 5 * values}
    return {"bytes": 2 * values * size + teacher + 8 * n, "flops": 12 * values}


# ---------------------------------------------------------------------------------------------------------------------
# inputs


def _layer(case):
    """Descriptors of a dense layer, as a program that calls the package keeps them."""
    import phoenix_core_b200 as pcb
    comps, ci, co = COMPONENTS[case["algebra"]], case["ci"], case["co"]
    algebra, layout = _algebra(case), {"io": pcb.FilterLayout.IO, "oi": pcb.FilterLayout.OI}[case["layout"]]
    ishape, fshape = (comps * case["n"], ci), _filter_shape(case)
    return {"fwd": pcb.DenseFwdDescriptor(ishape, fshape, algebra, layout, case["bias"]),
            "bwd": pcb.DenseBwdDescriptor(ishape, fshape, algebra, layout, True),
            "filter8": pcb.Filter8(fshape, algebra, layout, DEVICE)}


def _algebra(case):
    import phoenix_core_b200 as pcb
    return {"real": pcb.Algebra.REAL, "complex": pcb.Algebra.COMPLEX, "quaternion": pcb.Algebra.QUATERNION,
            "ga300": pcb.Algebra.GA_300}[case["algebra"]]


def _filter_shape(case):
    comps = COMPONENTS[case["algebra"]]
    shape = (case["ci"], case["co"]) if case["layout"] == "io" else (case["co"], case["ci"])
    return shape if comps == 1 else (comps,) + shape


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, comps, n = DTYPES[case["dtype"]], COMPONENTS[case["algebra"]], case["n"]

    def normal(shape, std=1.0):
        return torch.randn(shape, generator=gen, device=DEVICE).mul_(std)

    state = {"case": case, "dtype": dtype}
    if case["op"] == "dense8":
        ci, co = case["ci"], case["co"]
        # features of different sizes, as behind a trained norm
        state["x"] = (normal((comps * n, ci)) * normal((1, ci), 0.5).exp()).to(dtype)
        state["w"] = normal(_filter_shape(case), (1.0 / (comps * ci)) ** 0.5).to(dtype)
        state["bias"] = normal((co,) if comps == 1 else (comps, co), 0.1).to(dtype) if case["bias"] else None
        state["dy"] = (normal((comps * n, co)) * normal((1, co), 0.5).exp() * 2.0 ** -6).to(dtype) if case["mode"] == "train" else None
        if own:
            import phoenix_core_b200 as pcb
            state["layer"] = _layer(case)
            if case["mode"] == "fwd":
                pcb.quantizeFilter8(state["w"], state["layer"]["filter8"])
        elif case["mode"] == "fwd":
            # what a plain program keeps of the filter: e4m3 numbers and a scale for each block
            state["w8"] = _quantize(state["w"].float().view(comps, *state["w"].shape[-2:]), 128, 128)
        return state
    if case["op"] == "norm":
        features, gates = case["features"], case["gates"]
        state["x"] = (normal((comps * n, features)) * 2.0).to(dtype)
        state["branch"] = (normal((comps * n, features)) * normal((1, features), 0.5).exp()).to(dtype)
        state["gate"] = (1.0 + normal((comps * gates, features), 0.3)).to(dtype) if gates else None
        state["post"], state["pre"] = (1.0 + normal((features,), 0.1) for _ in range(2))
        if case["mode"] == "bwd":
            y, _, stats = _norm_forward(state)
            state["y"], state["stats"] = y.to(dtype), stats
            state["dy"], state["dh"] = (normal((comps * n, features), 2.0 ** -4).to(dtype) for _ in range(2))
        if own:
            import phoenix_core_b200 as pcb
            state["descriptor"] = pcb.ResidualNormDescriptor((comps * n, features), gates, _algebra(case), case["scale"], EPSILON)
        return state
    units, entries = case["units"], case["entries"]
    classes = comps * units
    steps = torch.randint(1, classes // entries + 1, (n, entries), generator=gen, device=DEVICE)
    index = steps.cumsum(1) - 1                                     # distinct, anywhere in the vocabulary
    teacher = normal((n, entries), 2.0).sort(dim=1, descending=True).values + 8.0
    logits = normal((n, classes), 1.5)
    logits.scatter_add_(1, index, 0.7 * teacher)
    logits = logits.to(dtype).view(n, comps, units).transpose(0, 1).reshape(comps * n, units)
    labels = index[:, 0].clone()                                    # mostly what the teacher says
    labels[::3] = torch.randint(0, classes, (n,), generator=gen, device=DEVICE)[::3]
    if case["holes"]:
        # rows without a label, rows with fewer entries than places, rows with none
        labels[::4] = -1
        cut = torch.randint(0, entries + 1, (n, 1), generator=gen, device=DEVICE)
        cut[1::5] = 0
        index = torch.where(torch.arange(entries, device=DEVICE) < cut, index, torch.full_like(index, -1))
    state.update(logits=logits.contiguous(), labels=labels, teacher=teacher.to(dtype), index=index)
    # the loss scale of the harness over the batch, with a weight for each sample
    state["grad"] = (0.5 + torch.rand((n,), generator=gen, device=DEVICE)) * (256.0 / n) if case["mode"] == "train" else None
    if own:
        import phoenix_core_b200 as pcb
        state["descriptor"] = pcb.DistillDescriptor(tuple(state["logits"].shape), entries, case["alpha"], case["temperature"], _algebra(case))
    return state


EPSILON = 1e-6


# ---------------------------------------------------------------------------------------------------------------------
# one pass


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    import phoenix_core_b200 as pcb
    case = state["case"]
    if case["op"] == "dense8":
        x, layer = state["x"], state["layer"]
        y = torch.empty(layer["fwd"].getOutputShape(), dtype=x.dtype, device=x.device)
        if case["mode"] == "fwd":
            pcb.dense8Fwd(x, layer["filter8"], state["bias"], y, layer["fwd"])
            return y
        pcb.quantizeFilter8(state["w"], layer["filter8"])
        pcb.dense8Fwd(x, layer["filter8"], None, y, layer["fwd"])
        dw = torch.empty(state["w"].shape[:-2] + (case["ci"], case["co"]), dtype=x.dtype, device=x.device)
        dx = torch.empty_like(x)
        pcb.dense8Bwd(x, layer["filter8"], state["dy"], dw, dx, layer["bwd"])
        return {"y": y, "dw": dw, "dx": dx}
    descriptor = state["descriptor"]
    if case["op"] == "norm":
        x, branch, gate, post, pre = (state[k] for k in ("x", "branch", "gate", "post", "pre"))
        if case["mode"] == "fwd":
            y, h = torch.empty_like(x), torch.empty_like(x)
            stats = torch.empty((2, case["n"]), dtype=torch.float32, device=x.device)
            pcb.residualNormFwd(x, branch, gate, post, pre, y, h, stats, descriptor)
            return {"y": y, "h": h, "stats": stats}
        dx, dbranch = torch.empty_like(x), torch.empty_like(x)
        dgate = None if gate is None else torch.empty_like(gate)
        dpost, dpre = torch.empty_like(post), torch.empty_like(pre)
        pcb.residualNormBwd(state["y"], branch, gate, post, pre, state["stats"], state["dy"], state["dh"],
                            dx, dbranch, dgate, dpost, dpre, descriptor)
        grads = {"dx": dx, "dbranch": dbranch, "dpost": dpost, "dpre": dpre}
        if gate is not None:
            grads["dgate"] = dgate
        return grads
    logits, teacher = state["logits"], state["teacher"]
    loss = torch.empty((case["n"],), dtype=torch.float32, device=logits.device)
    stats = torch.empty((3, case["n"]), dtype=torch.float32, device=logits.device)
    pcb.distillFwd(logits, state["labels"], teacher, state["index"], loss, stats, descriptor)
    if case["mode"] == "fwd":
        return loss
    dlogits = torch.empty_like(logits)
    pcb.distillBwd(logits, state["labels"], teacher, state["index"], stats, state["grad"], dlogits, descriptor)
    return {"loss": loss, "dlogits": dlogits}


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms


def _quantize(x, rows, cols):
    """e4m3 numbers and scales of the blocks of rows x cols of an fp32 [components, R, C]."""
    d, r, c = x.shape
    padded = torch.nn.functional.pad(x, (0, -c % cols, 0, -r % rows))
    blocks = padded.view(d, padded.shape[1] // rows, rows, padded.shape[2] // cols, cols)
    mantissa, exponent = torch.frexp(blocks.abs().amax(dim=(2, 4), keepdim=True))     # mantissa in [0.5, 1)
    exponent = exponent - 9 + (mantissa > 0.875).int()
    exponent = torch.where(mantissa == 0, torch.zeros_like(exponent), exponent).clamp_(min=-126)
    scale = ((exponent + 127) << 23).view(torch.float32)                              # 2^exponent exactly: pow() need not be
    return (blocks / scale).to(torch.float8_e4m3fn), scale, (r, c)


def _held(quantized):
    """The values that quantised blocks stand for."""
    q, scale, (r, c) = quantized
    v = q.float() * scale
    return v.reshape(v.shape[0], v.shape[1] * v.shape[2], -1)[:, :r, :c]


def _blades(algebra):
    return (0, 1, 2, 4, 3, 5, 6, 7) if algebra == "ga300" else tuple(range(COMPONENTS[algebra]))


def _terms(algebra):
    """(l, r, d, sign): component l of the input times component r of the filter adds to component d of the output."""
    bits = _blades(algebra)
    if algebra == "ga300":
        for l, a in enumerate(bits):
            for r, b in enumerate(bits):
                swaps = sum(bin((a >> s) & b).count("1") for s in (1, 2))
                yield l, r, bits.index(a ^ b), -1.0 if swaps % 2 else 1.0
        return
    minus = {"real": (), "complex": ((1, 1),), "quaternion": ((1, 1), (1, 3), (2, 1), (2, 2), (3, 2), (3, 3))}[algebra]
    for l in range(len(bits)):
        for r in range(len(bits)):
            yield l, r, l ^ r, -1.0 if (l, r) in minus else 1.0


def _run_plain(state):
    case, dtype = state["case"], state["dtype"]
    if case["op"] == "dense8":
        return _dense8_plain(state)
    if case["op"] == "norm":
        if case["mode"] == "fwd":
            y, h, stats = _norm_forward(state)
            return {"y": y.to(dtype), "h": h.to(dtype), "stats": stats}
        return _norm_backward(state)
    return _distill_plain(state)


def _dense8_plain(state):
    case, dtype, comps = state["case"], state["dtype"], COMPONENTS[state["case"]["algebra"]]
    x = state["x"].float().view(comps, case["n"], case["ci"])
    if case["mode"] == "fwd":
        w8 = state["w8"]
    else:
        w8 = _quantize(state["w"].float().view(comps, *state["w"].shape[-2:]), 128, 128)
    w = _held(w8)
    if case["layout"] == "oi":
        w = w.transpose(1, 2)
    xr = _held(_quantize(x, 1, 128))
    y = torch.zeros((comps, case["n"], case["co"]), device=x.device)
    for l, r, d, sign in _terms(case["algebra"]):
        y[d].addmm_(xr[l], w[r], alpha=sign)
    if state["bias"] is not None:
        y += state["bias"].float().view(comps, 1, case["co"])
    y = y.view(comps * case["n"], case["co"]).to(dtype)
    if case["mode"] == "fwd":
        return y
    dy = state["dy"].float().view(comps, case["n"], case["co"])
    dyr, dyc, xc = _held(_quantize(dy, 1, 128)), _held(_quantize(dy, 128, 1)), _held(_quantize(x, 128, 1))
    dx, dw = torch.zeros_like(x), torch.zeros((comps, case["ci"], case["co"]), device=x.device)
    for l, r, d, sign in _terms(case["algebra"]):
        dx[l].addmm_(dyr[d], w[r].t(), alpha=sign)
        dw[r].addmm_(xc[l].t(), dyc[d], alpha=sign)
    return {"y": y, "dw": dw.to(dtype).view(state["w"].shape[:-2] + (case["ci"], case["co"])), "dx": dx.view_as(state["x"]).to(dtype)}


def _samples(t, comps):
    """[components * n, f] as fp32 [n, components, f]."""
    return t.float().view(comps, -1, t.shape[1]).transpose(0, 1)


def _stacked(t, comps):
    return t.transpose(0, 1).reshape(comps * t.shape[0], t.shape[2])


def _gate(state):
    case, comps = state["case"], COMPONENTS[state["case"]["algebra"]]
    if state["gate"] is None:
        return 1.0
    return _samples(state["gate"], comps).repeat_interleave(case["n"] // case["gates"], dim=0)


def _norm_forward(state):
    case, comps = state["case"], COMPONENTS[state["case"]["algebra"]]
    x, b = _samples(state["x"], comps), _samples(state["branch"], comps)
    rb = torch.rsqrt(b.square().mean(dim=(1, 2), keepdim=True) + EPSILON)
    y = x + case["scale"] * _gate(state) * (b * rb * state["post"])
    ry = torch.rsqrt(y.square().mean(dim=(1, 2), keepdim=True) + EPSILON)
    h = y * ry * state["pre"]
    return _stacked(y, comps), _stacked(h, comps), torch.stack((rb.flatten(), ry.flatten()))


def _norm_backward(state):
    case, dtype, comps = state["case"], state["dtype"], COMPONENTS[state["case"]["algebra"]]
    y, b, dy, dh = (_samples(state[k], comps) for k in ("y", "branch", "dy", "dh"))
    rb, ry = state["stats"].view(2, -1, 1, 1)
    gate = _gate(state)
    yn, t = y * ry, dh * state["pre"]
    dpre = (dh * yn).sum(dim=(0, 1), dtype=torch.float64).float()
    dx = dy + ry * (t - yn * (t * yn).mean(dim=(1, 2), keepdim=True))
    u = b * rb
    dn = case["scale"] * gate * dx
    dpost = (dn * u).sum(dim=(0, 1), dtype=torch.float64).float()
    du = dn * state["post"]
    db = rb * (du - u * (du * u).mean(dim=(1, 2), keepdim=True))
    grads = {"dx": _stacked(dx, comps).to(dtype), "dbranch": _stacked(db, comps).to(dtype), "dpost": dpost, "dpre": dpre}
    if state["gate"] is not None:
        dgate = (case["scale"] * dx * u * state["post"]).view(case["gates"], -1, comps, case["features"]).sum(dim=1)
        grads["dgate"] = _stacked(dgate, comps).to(dtype)
    return grads


def _distill_plain(state):
    case, comps = state["case"], COMPONENTS[state["case"]["algebra"]]
    n, classes = case["n"], comps * case["units"]
    alpha, temperature = case["alpha"], case["temperature"]
    z = state["logits"].float().view(comps, n, case["units"]).transpose(0, 1).reshape(n, classes)
    labels, index = state["labels"], state["index"]
    top = z.amax(dim=1, keepdim=True)
    s1 = torch.exp(z - top).sum(dim=1, keepdim=True)
    st = torch.exp((z - top) / temperature).sum(dim=1, keepdim=True)
    has = ((labels >= 0) & (labels < classes)).float()[:, None]
    label = labels.clamp(0, classes - 1)[:, None]
    hard = has * (torch.log(s1) - (z.gather(1, label) - top))
    kept = (index >= 0) & (index < classes)
    places = index.clamp(0, classes - 1)
    t = torch.where(kept, state["teacher"].float() / temperature, torch.full_like(state["teacher"], float("-inf"), dtype=torch.float32))
    peak = t.amax(dim=1, keepdim=True)
    some = (peak > float("-inf")).float()
    shifted = torch.where(kept, t - torch.where(some > 0, peak, torch.zeros_like(peak)), t)
    e = torch.exp(shifted)
    total = e.sum(dim=1, keepdim=True)
    p = e / torch.where(some > 0, total, torch.ones_like(total))
    log_p = shifted - torch.log(total)
    log_q = (z.gather(1, places) - top) / temperature - torch.log(st)
    soft = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(dim=1, keepdim=True)
    loss = ((1.0 - alpha) * hard + alpha * temperature ** 2 * soft)[:, 0]
    if case["mode"] == "fwd":
        return loss
    dz = torch.exp(z - top) / s1 * ((1.0 - alpha) * has)
    dz.scatter_add_(1, label, -(1.0 - alpha) * has)
    dz += torch.exp((z - top) / temperature) / st * (alpha * temperature * some)
    dz.scatter_add_(1, places, -alpha * temperature * p)
    dz *= state["grad"][:, None]
    dz = dz.to(state["dtype"]).view(n, comps, case["units"]).transpose(0, 1).reshape(comps * n, case["units"])
    return {"loss": loss, "dlogits": dz.contiguous()}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    return {"dense8": _exact_dense8, "norm": _exact_norm, "distill": _exact_distill}[case["op"]](case, state)


def _power(e):
    """2^e of whole numbers in float64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(v):
    """The nearest e4m3 number, ties to the even one, of a float64 of magnitude 448 at most."""
    _, e = torch.frexp(v)
    step = _power(torch.clamp(e - 1, min=-6) - 3)
    return torch.round(v / step) * step


def _blockwise(x, axis):
    """x (float64, [components, R, C]) rounded in blocks of 128 along `axis`, or of 128 x 128 where it is None."""
    out = torch.empty_like(x)
    rows, cols = {1: (128, 1 << 30), 2: (1 << 30, 128), None: (128, 128)}[axis]
    for r in range(0, x.shape[1], rows):
        for c in range(0, x.shape[2], cols):
            block = x[:, r:r + rows, c:c + cols]
            top = block.abs().amax(dim=(1, 2) if axis is None else axis, keepdim=True)
            e = torch.floor(torch.log2(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448.0))
            e = torch.where(448.0 * _power(e) < top, e + 1, e)
            e = torch.where((top > 0) & (448.0 * _power(e - 1) >= top), e - 1, e).clamp(min=-126)
            out[:, r:r + rows, c:c + cols] = _round_e4m3(block / _power(e)) * _power(e)
    return out


def _exact_dense8(case, state):
    comps, n, ci, co = COMPONENTS[case["algebra"]], case["n"], case["ci"], case["co"]
    x = state["x"].double().view(comps, n, ci)
    w = _blockwise(state["w"].double().view(comps, *state["w"].shape[-2:]), None)
    if case["layout"] == "oi":
        w = w.transpose(1, 2)
    # the product as one real matrix of components x components blocks
    big = torch.zeros((comps, ci, comps, co), dtype=torch.float64, device=x.device)
    terms = list(_terms(case["algebra"]))
    for l, r, d, sign in terms:
        big[l, :, d] = sign * w[r]
    big = big.view(comps * ci, comps * co)

    def wide(t):
        return t.transpose(0, 1).reshape(n, -1)

    def tall(t, features):
        return t.view(n, comps, features).transpose(0, 1).reshape(comps * n, features)

    y = wide(_blockwise(x, 2)) @ big
    if state["bias"] is not None:
        y = y + state["bias"].double().flatten()
    y = tall(y, co)
    if case["mode"] == "fwd":
        return y
    dy = state["dy"].double().view(comps, n, co)
    dx = tall(wide(_blockwise(dy, 2)) @ big.t(), ci)
    outer = (wide(_blockwise(x, 1)).t() @ wide(_blockwise(dy, 1))).view(comps, ci, comps, co)
    dw = torch.zeros((comps, ci, co), dtype=torch.float64, device=x.device)
    for l, r, d, sign in terms:
        dw[r] += sign * outer[l, :, d]
    return {"y": y, "dw": dw.view(state["w"].shape[:-2] + (ci, co)), "dx": dx}


def _exact_norm(case, state):
    comps, n, f = COMPONENTS[case["algebra"]], case["n"], case["features"]

    def wide(t):
        return t.double().view(comps, -1, f).transpose(0, 1).reshape(-1, comps * f)

    def tall(t):
        return t.view(-1, comps, f).transpose(0, 1).reshape(-1, f)

    b, scale = wide(state["branch"]), float(case["scale"])
    post, pre = state["post"].double().repeat(comps), state["pre"].double().repeat(comps)
    gate = torch.ones((1, comps * f), dtype=torch.float64, device=b.device) if state["gate"] is None else wide(state["gate"])
    groups = gate.shape[0]
    gate = gate[torch.arange(n, device=b.device) // (n // groups)]
    if case["mode"] == "fwd":
        rb = 1.0 / torch.sqrt((b * b).sum(dim=1) / (comps * f) + EPSILON)
        y = wide(state["x"]) + scale * gate * post * b * rb[:, None]
        ry = 1.0 / torch.sqrt((y * y).sum(dim=1) / (comps * f) + EPSILON)
        return {"y": tall(y), "h": tall(pre * y * ry[:, None]), "stats": torch.stack((rb, ry))}
    y, dy, dh = wide(state["y"]), wide(state["dy"]), wide(state["dh"])
    rb, ry = state["stats"].double()
    ry, rb = ry[:, None], rb[:, None]
    # d(y * ry)/dy = ry * I - ry^3 / width * y y^T, and the same for the branch
    g = dh * pre
    dx = dy + ry * g - ry ** 3 / (comps * f) * y * (g * y).sum(dim=1, keepdim=True)
    dnormed = scale * gate * dx
    v = dnormed * post
    db = rb * v - rb ** 3 / (comps * f) * b * (v * b).sum(dim=1, keepdim=True)
    grads = {"dx": tall(dx), "dbranch": tall(db), "dpost": (dnormed * b * rb).sum(dim=0).view(comps, f).sum(dim=0),
             "dpre": (dh * y * ry).sum(dim=0).view(comps, f).sum(dim=0)}
    if state["gate"] is not None:
        grads["dgate"] = tall((scale * dx * post * b * rb).view(groups, n // groups, comps * f).sum(dim=1))
    return grads


def _exact_distill(case, state):
    comps, n, units = COMPONENTS[case["algebra"]], case["n"], case["units"]
    classes, alpha, temp = comps * units, float(case["alpha"]), float(case["temperature"])
    logits = state["logits"].view(comps, n, units)
    losses, grads = [], []
    rows = max(1, (1 << 26) // classes)
    for first in range(0, n, rows):
        z = logits[:, first:first + rows].double().transpose(0, 1).reshape(-1, classes)
        labels, index = state["labels"][first:first + rows], state["index"][first:first + rows]
        t = state["teacher"][first:first + rows].double() / temp
        log1, logt = torch.log_softmax(z, dim=1), torch.log_softmax(z / temp, dim=1)
        valid = (labels >= 0) & (labels < classes)
        place = torch.where(valid, labels, torch.zeros_like(labels))[:, None]
        hard = torch.where(valid, -log1.gather(1, place)[:, 0], torch.zeros_like(log1[:, 0]))
        inside = (index >= 0) & (index < classes)
        where = torch.where(inside, index, torch.zeros_like(index))
        t = t.masked_fill(~inside, float("-inf"))
        log_p = torch.log_softmax(t, dim=1)
        p = torch.where(t > float("-inf"), log_p.exp(), torch.zeros_like(t))
        some = inside.any(dim=1)
        soft = torch.where(p > 0, p * (log_p - logt.gather(1, where)), torch.zeros_like(p)).sum(dim=1)
        losses.append((1.0 - alpha) * hard + alpha * temp * temp * soft)
        if case["mode"] == "train":
            dz = (1.0 - alpha) * valid.double()[:, None] * log1.exp() + alpha * temp * some.double()[:, None] * logt.exp()
            dz.scatter_add_(1, place, -(1.0 - alpha) * valid.double()[:, None])
            dz.scatter_add_(1, where, -alpha * temp * p)
            grads.append(dz * state["grad"][first:first + rows].double()[:, None])
    loss = torch.cat(losses)
    if case["mode"] == "fwd":
        return loss
    dz = torch.cat(grads).view(n, comps, units).transpose(0, 1).reshape(comps * n, units)
    return {"loss": loss, "dlogits": dz}
