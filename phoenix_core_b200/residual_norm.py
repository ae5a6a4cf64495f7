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
from .ops import _ALGEBRAS, _DTYPES, Device, _launch, _need, _need_input


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
        self.gateShape, self.weightShape, self.statsShape = (dim * self.gateRows, self.inputShape[1]), (self.inputShape[1],), (2, self.samples)
        self._calls = {}

    def getInputShape(self): return self.inputShape
    def getGateShape(self): return self.gateShape
    def getWeightShape(self): return self.weightShape
    def getStatsShape(self): return self.statsShape
    def getAlgebra(self): return self.algebra

    def _call(self, dtype):
        call = self._calls.get(dtype)
        if call is None:
            d = _lib.NormDesc()
            d.dtype, d.algebra, d.batch, d.features = _DTYPES[dtype], _ALGEBRAS[self.algebra], self.samples, self.inputShape[1]
            d.gate_rows, d.residual_scale, d.epsilon = self.gateRows, self.residualScale, self.epsilon
            ref = ctypes.byref(d)
            call = self._calls[dtype] = (ref, _lib.lib().pcb_residual_norm_bwd_workspace_size(ref))
        return call


def _check_parts(descriptor, dtype, index, branch, gate, post, pre):
    if branch is not None:
        _need(branch, "branch", dtype, descriptor.inputShape, index)
    elif gate is not None or post is not None:
        raise ValueError("a gate or postWeight without a branch")
    if (gate is None) != (descriptor.gateRows == 0):
        raise ValueError("the descriptor has %d rows of a gate" % descriptor.gateRows)
    if gate is not None:
        _need(gate, "gate", dtype, descriptor.gateShape, index)
    if post is not None:
        _need(post, "postWeight", torch.float32, descriptor.weightShape, index)
    if pre is not None:
        _need(pre, "preWeight", torch.float32, descriptor.weightShape, index)


def _ptr(t):
    return None if t is None else t.data_ptr()


def residualNormFwd(residualTensor, branchTensor, gateTensor, postWeight, preWeight, outputTensor, normTensor, statsTensor, descriptor):
    """y into ``outputTensor`` and h into ``normTensor``; ``statsTensor`` (fp32, ``getStatsShape()``) keeps the factors of both norms for the
    backward call and may be None. Without a branch (None, with gate and postWeight) h is the norm of the residual itself and
    ``outputTensor`` may be None; without ``normTensor`` (None, with preWeight) there is no norm behind the block. Weights may be None (ones)."""
    x, dtype = residualTensor, residualTensor.dtype
    shape = descriptor.inputShape
    index = _need_input(x, "residual", shape)
    _check_parts(descriptor, dtype, index, branchTensor, gateTensor, postWeight, preWeight)
    if (branchTensor is not None or normTensor is None) and outputTensor is None:
        raise ValueError("output expected")
    if outputTensor is not None:
        _need(outputTensor, "output", dtype, shape, index)
    if normTensor is not None:
        _need(normTensor, "norm", dtype, shape, index)
    elif preWeight is not None:
        raise ValueError("preWeight without normTensor")
    if statsTensor is not None:
        _need(statsTensor, "stats", torch.float32, descriptor.statsShape, index)
    if shape[0] == 0:
        return
    _launch(index, _lib.lib().pcb_residual_norm_fwd, descriptor._call(dtype)[0], x.data_ptr(), _ptr(branchTensor), _ptr(gateTensor), _ptr(postWeight),
            _ptr(preWeight), _ptr(outputTensor), _ptr(normTensor), _ptr(statsTensor))


def residualNormBwd(outputTensor, branchTensor, gateTensor, postWeight, preWeight, statsTensor, gradOutput, gradNorm, gradResidual, gradBranch,
                    gradGate, gradPostWeight, gradPreWeight, descriptor):
    """From ``gradOutput`` (of y, from the residual path; None: none) and ``gradNorm`` (of h; None: there was no norm behind the block) the
    gradients of the residual, the branch, the gate and the weights; those of the gate and the weights may be None. ``outputTensor`` is the forward
    call's y (the residual itself where there was no branch), needed where there is a ``gradNorm``."""
    dtype, shape, weights = gradResidual.dtype, descriptor.inputShape, descriptor.weightShape
    index = _need_input(gradResidual, "gradResidual", shape)
    _check_parts(descriptor, dtype, index, branchTensor, gateTensor, postWeight, preWeight)
    if gradOutput is None and gradNorm is None:
        raise ValueError("gradOutput or gradNorm expected")
    if gradNorm is None:
        if preWeight is not None or gradPreWeight is not None:
            raise ValueError("preWeight without gradNorm")
    else:
        if outputTensor is None:
            raise ValueError("output expected: the gradient of its norm needs it")
        _need(gradNorm, "gradNorm", dtype, shape, index)
        _need(outputTensor, "output", dtype, shape, index)
    if gradOutput is not None:
        _need(gradOutput, "gradOutput", dtype, shape, index)
    if branchTensor is not None:
        if gradBranch is None:
            raise ValueError("gradBranch expected")
        _need(gradBranch, "gradBranch", dtype, shape, index)
    elif gradPostWeight is not None:
        raise ValueError("gradPostWeight without a branch")
    if gradGate is not None:
        if gateTensor is None:
            raise ValueError("gradGate without a gate")
        _need(gradGate, "gradGate", dtype, descriptor.gateShape, index)
    if gradPostWeight is not None:
        _need(gradPostWeight, "gradPostWeight", torch.float32, weights, index)
    if gradPreWeight is not None:
        _need(gradPreWeight, "gradPreWeight", torch.float32, weights, index)
    if statsTensor is None:
        raise ValueError("stats expected")
    _need(statsTensor, "stats", torch.float32, descriptor.statsShape, index)
    if shape[0] == 0:
        for t in (gradPostWeight, gradPreWeight, gradGate):
            if t is not None:
                t.zero_()
        return
    ref, need = descriptor._call(dtype)
    dev = Device.at(index)
    with dev.accessControl:
        ws = dev.requestWorkspace(need + 256)                          # behind the workspace's status block
        _launch(index, _lib.lib().pcb_residual_norm_bwd, ref, _ptr(outputTensor), _ptr(branchTensor), _ptr(gateTensor), _ptr(postWeight), _ptr(preWeight),
                statsTensor.data_ptr(), _ptr(gradOutput), _ptr(gradNorm), gradResidual.data_ptr(), _ptr(gradBranch), _ptr(gradGate), _ptr(gradPostWeight),
                _ptr(gradPreWeight), ws.data_ptr() + 256, ws.numel() - 256)
