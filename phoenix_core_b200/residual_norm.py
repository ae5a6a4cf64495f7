"""The norms before and after a residual block, with the block's gate and residual scale, each direction in one pass over the
data: ``residualNormFwd`` and ``residualNormBwd`` (no counterpart in the reference, which has no normalisation).

A sample is all of its components' features, stacked on the leading axis as in every tensor of the engine:

    n(v) = v / sqrt(mean(v^2) + epsilon)
    y = x + residualScale * gate * (n(branch) * postWeight)         the block's output behind its norm, joined to the residual path
    h = n(y) * preWeight                                            what the next block reads

The weights are fp32, one per feature and shared by its components (as the gamma of the batch-norm helpers is); the mean runs over all components,
so that a norm scales a sample and keeps the directions of its quaternions. A gate holds a factor for each value of a group of consecutive
samples: ``gateRows`` of them, from one for all samples to one for each.
"""
import ctypes

import torch

from . import _lib
from .descriptors import MULTIVECTOR_DIM, Algebra
from .ops import _ALGEBRAS, _DTYPES, Device, _check_tensor, _OnDevice, _ptr, _stream


class ResidualNormDescriptor:
    """``inputShape``: (components * samples, features); ``gateRows``: rows of the gate per component, a divisor of the samples (0: no gate)."""

    def __init__(self, inputShape, gateRows=0, algebra=Algebra.REAL, residualScale=1.0, epsilon=1e-6):
        self.inputShape = tuple(int(s) for s in inputShape)
        self.gateRows, self.algebra, self.residualScale, self.epsilon = int(gateRows), algebra, float(residualScale), float(epsilon)
        dim = MULTIVECTOR_DIM[algebra]
        if len(self.inputShape) != 2 or self.inputShape[1] <= 0 or self.inputShape[0] % dim != 0:
            raise ValueError("input shape %s: (components * samples, features) expected, with %d components" % (self.inputShape, dim))
        self.samples = self.inputShape[0] // dim
        if self.gateRows < 0 or (self.gateRows > 0 and self.samples % self.gateRows != 0):
            raise ValueError("%d rows of the gate for %d samples" % (self.gateRows, self.samples))
        if not self.epsilon >= 0.0:
            raise ValueError("epsilon must not be negative")
        self._desc = {}

    def getInputShape(self): return self.inputShape
    def getGateShape(self): return (MULTIVECTOR_DIM[self.algebra] * self.gateRows, self.inputShape[1])
    def getWeightShape(self): return (self.inputShape[1],)
    def getStatsShape(self): return (2, self.samples)
    def getAlgebra(self): return self.algebra

    def _c(self, dtype):
        d = self._desc.get(dtype)
        if d is None:
            d = _lib.NormDesc()
            d.dtype, d.algebra, d.batch, d.features = _DTYPES[dtype], _ALGEBRAS[self.algebra], self.samples, self.inputShape[1]
            d.gate_rows, d.residual_scale, d.epsilon = self.gateRows, self.residualScale, self.epsilon
            self._desc[dtype] = d
        return d


def _check_optional(t, name, like, shape, dtype=None):
    if t is not None:
        _check_tensor(t, name, like.dtype if dtype is None else dtype, shape)
        if t.device != like.device:
            raise ValueError("%s is on %s, the input on %s" % (name, t.device, like.device))


def _check_first(t, name, descriptor):
    if t.dtype not in _DTYPES:
        raise ValueError("%s dtype %s: float32, float16 or bfloat16 expected" % (name, t.dtype))
    _check_tensor(t, name, shape=descriptor.getInputShape())


def _check_parts(descriptor, like, branch, gate, post, pre):
    shape, weights = descriptor.getInputShape(), descriptor.getWeightShape()
    _check_optional(branch, "branch", like, shape)
    if (gate is None) != (descriptor.gateRows == 0):
        raise ValueError("the descriptor has %d rows of a gate" % descriptor.gateRows)
    _check_optional(gate, "gate", like, descriptor.getGateShape())
    _check_optional(post, "postWeight", like, weights, torch.float32)
    _check_optional(pre, "preWeight", like, weights, torch.float32)
    if branch is None and (gate is not None or post is not None):
        raise ValueError("a gate or postWeight without a branch")


def residualNormFwd(residualTensor, branchTensor, gateTensor, postWeight, preWeight, outputTensor, normTensor, statsTensor, descriptor):
    """y into ``outputTensor`` and h into ``normTensor``; ``statsTensor`` (fp32, ``getStatsShape()``) keeps the factors of both norms for the
    backward call and may be None. Without a branch (None, with gate and postWeight) h is the norm of the residual itself and
    ``outputTensor`` may be None; without ``normTensor`` (None, with preWeight) there is no norm behind the block. Weights may be None (ones)."""
    x = residualTensor
    _check_first(x, "residual", descriptor)
    _check_parts(descriptor, x, branchTensor, gateTensor, postWeight, preWeight)
    if (branchTensor is not None and outputTensor is None) or (outputTensor is None and normTensor is None):
        raise ValueError("output expected")
    if normTensor is None and preWeight is not None:
        raise ValueError("preWeight without normTensor")
    _check_optional(outputTensor, "output", x, x.shape)
    _check_optional(normTensor, "norm", x, x.shape)
    _check_optional(statsTensor, "stats", x, descriptor.getStatsShape(), torch.float32)
    if x.numel() == 0:
        return
    d = descriptor._c(x.dtype)
    dev = Device.get(x.device)
    with _OnDevice(dev.index):
        _lib.check(_lib.lib().pcb_residual_norm_fwd(ctypes.byref(d), _ptr(x), _ptr(branchTensor), _ptr(gateTensor), _ptr(postWeight), _ptr(preWeight),
                                                    _ptr(outputTensor), _ptr(normTensor), _ptr(statsTensor), _stream()))


def residualNormBwd(outputTensor, branchTensor, gateTensor, postWeight, preWeight, statsTensor, gradOutput, gradNorm, gradResidual, gradBranch,
                    gradGate, gradPostWeight, gradPreWeight, descriptor):
    """From ``gradOutput`` (of y, from the residual path; None: none) and ``gradNorm`` (of h; None: there was no norm behind the block) the
    gradients of the residual, the branch, the gate and the weights; those of the gate and the weights may be None. ``outputTensor`` is the forward
    call's y (the residual itself where there was no branch), needed where there is a ``gradNorm``."""
    like = gradResidual
    _check_first(like, "gradResidual", descriptor)
    _check_parts(descriptor, like, branchTensor, gateTensor, postWeight, preWeight)
    shape, weights = descriptor.getInputShape(), descriptor.getWeightShape()
    if gradOutput is None and gradNorm is None:
        raise ValueError("gradOutput or gradNorm expected")
    if gradNorm is not None and outputTensor is None:
        raise ValueError("output expected: the gradient of its norm needs it")
    if gradNorm is None and (preWeight is not None or gradPreWeight is not None):
        raise ValueError("preWeight without gradNorm")
    if branchTensor is None and gradPostWeight is not None:
        raise ValueError("gradPostWeight without a branch")
    if (gradGate is not None and gateTensor is None) or (branchTensor is not None and gradBranch is None):
        raise ValueError("gradGate without a gate, or a branch without gradBranch")
    for t, name in ((outputTensor, "output"), (gradOutput, "gradOutput"), (gradNorm, "gradNorm"), (gradBranch, "gradBranch")):
        _check_optional(t, name, like, shape)
    _check_optional(gradGate, "gradGate", like, descriptor.getGateShape())
    _check_optional(gradPostWeight, "gradPostWeight", like, weights, torch.float32)
    _check_optional(gradPreWeight, "gradPreWeight", like, weights, torch.float32)
    if statsTensor is None:
        raise ValueError("stats expected")
    _check_optional(statsTensor, "stats", like, descriptor.getStatsShape(), torch.float32)
    if like.numel() == 0:
        for t in (gradPostWeight, gradPreWeight, gradGate):
            if t is not None:
                t.zero_()
        return
    d = descriptor._c(like.dtype)
    L, dev = _lib.lib(), Device.get(like.device)
    with dev.accessControl, _OnDevice(dev.index):
        need = getattr(d, "_bwd_need", None)
        if need is None:
            need = d._bwd_need = L.pcb_residual_norm_bwd_workspace_size(ctypes.byref(d))
        ws = dev.requestWorkspace(need + 256)                          # behind the workspace's status block
        _lib.check(L.pcb_residual_norm_bwd(ctypes.byref(d), _ptr(outputTensor), _ptr(branchTensor), _ptr(gateTensor), _ptr(postWeight),
                                           _ptr(preWeight), _ptr(statsTensor), _ptr(gradOutput), _ptr(gradNorm), _ptr(gradResidual),
                                           _ptr(gradBranch), _ptr(gradGate), _ptr(gradPostWeight), _ptr(gradPreWeight),
                                           _ptr(ws) + 256, ws.numel() - 256, _stream()))
