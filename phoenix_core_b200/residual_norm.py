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
from .ops import _ALGEBRAS, _DTYPES, Device, _Entry, _input_device


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
            row, gate = (dtype, self.inputShape), (dtype, self.gateShape)
            weight, stats = (torch.float32, self.weightShape), (torch.float32, self.statsShape)
            block = [("branch",) + row, ("gate",) + gate, ("postWeight",) + weight, ("preWeight",) + weight]
            fwd = _Entry("pcb_residual_norm_fwd", d, [("residual",) + row] + block + [("output",) + row, ("norm",) + row, ("stats",) + stats])
            bwd = _Entry("pcb_residual_norm_bwd", d, [("output",) + row] + block + [
                ("stats",) + stats, ("gradOutput",) + row, ("gradNorm",) + row, ("gradResidual",) + row, ("gradBranch",) + row, ("gradGate",) + gate,
                ("gradPostWeight",) + weight, ("gradPreWeight",) + weight])
            call = self._calls[dtype] = (fwd, bwd, _lib.lib().pcb_residual_norm_bwd_workspace_size(ctypes.byref(d)))
        return call


def _check_parts(descriptor, branch, gate, post):
    if (gate is None) != (descriptor.gateRows == 0):
        raise ValueError("the descriptor has %d rows of a gate" % descriptor.gateRows)
    if branch is None and (gate is not None or post is not None):
        raise ValueError("a gate or postWeight without a branch")


def residualNormFwd(residualTensor, branchTensor, gateTensor, postWeight, preWeight, outputTensor, normTensor, statsTensor, descriptor):
    """y into ``outputTensor`` and h into ``normTensor``; ``statsTensor`` (fp32, ``getStatsShape()``) keeps the factors of both norms for the
    backward call and may be None. Without a branch (None, with gate and postWeight) h is the norm of the residual itself and
    ``outputTensor`` may be None; without ``normTensor`` (None, with preWeight) there is no norm behind the block. Weights may be None (ones)."""
    _input_device(residualTensor, "residual")
    _check_parts(descriptor, branchTensor, gateTensor, postWeight)
    if (branchTensor is not None or normTensor is None) and outputTensor is None:
        raise ValueError("output expected")
    if normTensor is None and preWeight is not None:
        raise ValueError("preWeight without normTensor")
    fwd = descriptor._call(residualTensor.dtype)[0]
    operands = (residualTensor, branchTensor, gateTensor, postWeight, preWeight, outputTensor, normTensor, statsTensor)
    if descriptor.samples:
        fwd.call(None, 0, *operands)
    else:
        fwd.check(*operands)


def residualNormBwd(outputTensor, branchTensor, gateTensor, postWeight, preWeight, statsTensor, gradOutput, gradNorm, gradResidual, gradBranch,
                    gradGate, gradPostWeight, gradPreWeight, descriptor):
    """From ``gradOutput`` (of y, from the residual path; None: none) and ``gradNorm`` (of h; None: there was no norm behind the block) the
    gradients of the residual, the branch, the gate and the weights; those of the gate and the weights may be None. ``outputTensor`` is the forward
    call's y (the residual itself where there was no branch), needed where there is a ``gradNorm``."""
    index = _input_device(gradResidual, "gradResidual")
    _check_parts(descriptor, branchTensor, gateTensor, postWeight)
    if gradOutput is None and gradNorm is None:
        raise ValueError("gradOutput or gradNorm expected")
    if gradNorm is None:
        if preWeight is not None or gradPreWeight is not None:
            raise ValueError("preWeight without gradNorm")
    elif outputTensor is None:
        raise ValueError("output expected: the gradient of its norm needs it")
    if branchTensor is None:
        if gradPostWeight is not None:
            raise ValueError("gradPostWeight without a branch")
    elif gradBranch is None:
        raise ValueError("gradBranch expected")
    if gradGate is not None and gateTensor is None:
        raise ValueError("gradGate without a gate")
    if statsTensor is None:
        raise ValueError("stats expected")
    _, bwd, need = descriptor._call(gradResidual.dtype)
    operands = (outputTensor, branchTensor, gateTensor, postWeight, preWeight, statsTensor, gradOutput, gradNorm, gradResidual, gradBranch, gradGate, gradPostWeight,
                gradPreWeight)
    if descriptor.samples == 0:
        bwd.check(*operands)
        for t in (gradPostWeight, gradPreWeight, gradGate):
            if t is not None:
                t.zero_()
        return
    dev = Device.at(index)
    with dev.accessControl:
        ws = dev.requestWorkspace(need)
        bwd.call(ws, 0, *operands)
        dev._after_op()
