"""What the block norms and the distillation refuse, without a GPU."""
import ctypes

import pytest
import torch

import phoenix_core_b200 as pcb
from phoenix_core_b200 import _lib

Q, R = pcb.Algebra.QUATERNION, pcb.Algebra.REAL


@pytest.fixture(scope="module")
def library():
    from phoenix_core_b200.csrc import build
    build.build()
    return _lib.lib()


def norm(batch=12, features=64, gates=3, dtype=_lib.PCB_F16, algebra=0, eps=1e-6):
    d = _lib.NormDesc()
    d.dtype, d.algebra, d.batch, d.features, d.gate_rows, d.residual_scale, d.epsilon = dtype, algebra, batch, features, gates, 1.0, eps
    return d


def distill(batch=4, units=250, entries=8, alpha=0.5, temperature=2.0, dtype=_lib.PCB_F16, algebra=0):
    d = _lib.DistillDesc()
    d.dtype, d.algebra, d.batch, d.units, d.entries, d.alpha, d.temperature = dtype, algebra, batch, units, entries, alpha, temperature
    return d


def test_norm_entry_points(library):
    p, bad = 1 << 20, _lib.PCB_ERR_INVALID_ARGUMENT                  # (never read: every call is refused before a launch)

    def fwd(d, x=p, b=p, g=p, post=p, pre=p, y=p, h=p):
        return library.pcb_residual_norm_fwd(ctypes.byref(d), x, b, g, post, pre, y, h, p, None)

    assert fwd(norm(), x=None) == bad and fwd(norm(), y=None) == bad and fwd(norm(), g=None) == bad and fwd(norm(gates=0)) == bad
    assert fwd(norm(), b=None) == bad and fwd(norm(gates=0), b=None, g=None) == bad and fwd(norm(), h=None) == bad
    assert fwd(norm(gates=5)) == bad and fwd(norm(gates=-1)) == bad and fwd(norm(features=0)) == bad and fwd(norm(dtype=9)) == bad
    assert fwd(norm(algebra=9)) == bad and fwd(norm(eps=-1.0)) == bad and fwd(norm(eps=float("nan"))) == bad
    assert fwd(norm(batch=1 << 20, gates=1, features=1 << 12)) == _lib.PCB_ERR_TOO_LARGE
    assert library.pcb_residual_norm_fwd(None, p, p, p, p, p, p, p, p, None) == bad
    assert fwd(norm(batch=0), x=None) == _lib.PCB_OK

    d = norm()
    need = library.pcb_residual_norm_bwd_workspace_size(ctypes.byref(d))
    assert need > 0 and library.pcb_residual_norm_bwd_workspace_size(ctypes.byref(norm(gates=5))) == 0

    def bwd(y=p, b=p, g=p, post=p, pre=p, stats=p, dy=p, dh=p, dx=p, db=p, dg=p, dpost=p, dpre=p, ws=p, size=need):
        return library.pcb_residual_norm_bwd(ctypes.byref(d), y, b, g, post, pre, stats, dy, dh, dx, db, dg, dpost, dpre, ws, size, None)

    assert bwd(size=need - 1) == _lib.PCB_ERR_WORKSPACE and bwd(ws=None) == _lib.PCB_ERR_WORKSPACE and bwd(ws=p + 4) == bad
    assert bwd(stats=None) == bad and bwd(dx=None) == bad and bwd(db=None) == bad and bwd(y=None) == bad and bwd(dy=None, dh=None) == bad
    assert bwd(dh=None) == bad and bwd(b=None) == bad and bwd(g=None) == bad


def test_distill_entry_points(library):
    p, bad = 1 << 20, _lib.PCB_ERR_INVALID_ARGUMENT

    def fwd(d, z=p, t=p, i=p, loss=p):
        return library.pcb_distill_fwd(ctypes.byref(d), z, p, t, i, loss, p, None)

    assert fwd(distill(), z=None) == bad and fwd(distill(), t=None) == bad and fwd(distill(), i=None) == bad and fwd(distill(), loss=None) == bad
    for wrong in (dict(units=0), dict(entries=-1), dict(alpha=1.5), dict(alpha=float("nan")), dict(temperature=0.0), dict(temperature=float("inf")), dict(dtype=5), dict(algebra=4)):
        assert fwd(distill(**wrong)) == bad, wrong
    assert fwd(distill(entries=5000)) == _lib.PCB_ERR_UNSUPPORTED
    assert fwd(distill(units=1 << 30)) == _lib.PCB_ERR_TOO_LARGE
    assert fwd(distill(batch=0), z=None) == _lib.PCB_OK
    d = distill()
    assert library.pcb_distill_bwd(ctypes.byref(d), p, p, p, p, p, p, p, None) == bad                  # in place
    assert library.pcb_distill_bwd(ctypes.byref(d), p, p, p, p, None, p, 2 * p, None) == bad
    assert library.pcb_distill_bwd(ctypes.byref(d), p, p, p, p, p, None, 2 * p, None) == bad


def test_norm_python():
    with pytest.raises(ValueError):
        pcb.ResidualNormDescriptor((7, 8), 0, Q)
    with pytest.raises(ValueError):
        pcb.ResidualNormDescriptor((8, 8), 3, R)
    with pytest.raises(ValueError):
        pcb.ResidualNormDescriptor((8, 8), 0, R, 1.0, -1.0)
    d = pcb.ResidualNormDescriptor((8, 16), 2, Q)
    assert d.getGateShape() == (8, 16) and d.getStatsShape() == (2, 2) and d.getWeightShape() == (16,)
    x = torch.zeros(8, 16)
    with pytest.raises(ValueError, match="CUDA"):
        pcb.residualNormFwd(x, x, x, None, None, x, x, None, d)
    with pytest.raises(ValueError):
        pcb.residualNormFwd(torch.zeros(8, 16, dtype=torch.float64), x, x, None, None, x, x, None, d)


def test_distill_python():
    for wrong in (dict(alpha=-0.1), dict(temperature=0.0), dict(teacherEntries=-1), dict(logitsShape=(7, 8))):
        with pytest.raises(ValueError):
            pcb.DistillDescriptor(**{**dict(logitsShape=(8, 250), teacherEntries=3, alpha=0.5, temperature=1.0, algebra=Q), **wrong})
    d = pcb.DistillDescriptor((8, 250), 3, 0.5, 2.0, Q)
    assert d.getClasses() == 1000 and d.getTeacherShape() == (2, 3) and d.getStatsShape() == (3, 2)
    with pytest.raises(ValueError, match="CUDA"):
        pcb.distillFwd(torch.zeros(8, 250), None, None, None, torch.zeros(2), None, d)


def test_results_apart(library):
    """A result on an operand, on another result, or across the end of one is refused (addresses are only compared: nothing is launched)."""
    bad, step = _lib.PCB_ERR_INVALID_ARGUMENT, 1 << 20
    at = [step * (i + 1) for i in range(16)]
    x, b, g, post, pre, y, h, stats = at[:8]
    row = 4 * 12 * 64 * 2                                            # bytes of the descriptor's rows
    for y_, h_, stats_ in ((x, h, stats), (y, b, stats), (y, y, stats), (x + row - 2, h, stats), (y, h, y), (g, h, stats), (y, pre, stats), (y, h, post)):
        assert library.pcb_residual_norm_fwd(ctypes.byref(norm()), x, b, g, post, pre, y_, h_, stats_, None) == bad
        assert b"shares memory" in library.pcb_last_error_message()
    need = library.pcb_residual_norm_bwd_workspace_size(ctypes.byref(norm()))
    dy, dh, dx, db, dg, dpost, dpre, ws = at[8:]
    for results in ((dy, db, dg, dpost, dpre), (dh, db, dg, dpost, dpre), (dx, dx, dg, dpost, dpre), (dx, b, dg, dpost, dpre), (dx, db, g, dpost, dpre), (dx, db, dg, post, dpre),
                    (dx, db, dg, dpost, dpost), (y, db, dg, dpost, dpre), (dx, db, dg, dpost, ws)):
        assert library.pcb_residual_norm_bwd(ctypes.byref(norm()), y, b, g, post, pre, stats, dy, dh, *results, ws, need, None) == bad
        assert b"shares memory" in library.pcb_last_error_message()
    d = _lib.DenseDesc()
    d.dtype, d.algebra, d.batch, d.in_features, d.out_features = _lib.PCB_F16, 0, 2, 128, 128
    need = library.pcb_qdense8_fwd_workspace_size(ctypes.byref(d))
    assert library.pcb_qdense8_fwd(ctypes.byref(d), x, b, g, None, x + 16, ws, need, None) == bad and b"share memory" in library.pcb_last_error_message()
