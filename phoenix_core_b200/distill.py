"""Distillation from a teacher's largest logits, mixed with the cross-entropy of the labels: ``distillFwd`` and ``distillBwd`` (no
counterpart in the reference, whose plugin leaves losses to the framework).

The logits are what a dense layer writes: ``[components * samples, units]``, class = component * units + unit. With p the softmax of
the teacher's logits over the classes that it names, and q the softmax of the student's over all, both at temperature T:

    loss = (1 - alpha) * crossEntropy(logits, label) + alpha * T^2 * sum_i p_i (log p_i - log q_i)

one number for each sample; a mean or a weighting is the caller's, through the gradient of the losses.
"""
import ctypes

import torch

from . import _lib
from .descriptors import MULTIVECTOR_DIM, Algebra
from .ops import _ALGEBRAS, _DTYPES, _Entry, _input_device


class DistillDescriptor:
    """``logitsShape``: (components * samples, units); ``teacherEntries``: classes that the teacher names per sample (0: labels only)."""

    def __init__(self, logitsShape, teacherEntries, alpha=0.5, temperature=1.0, algebra=Algebra.QUATERNION):
        self.logitsShape = tuple(int(s) for s in logitsShape)
        self.teacherEntries, self.alpha, self.temperature, self.algebra = int(teacherEntries), float(alpha), float(temperature), algebra
        dim = MULTIVECTOR_DIM[algebra]
        if len(self.logitsShape) != 2 or self.logitsShape[1] <= 0 or self.logitsShape[0] % dim != 0:
            raise ValueError("logits shape %s: (components * samples, units) expected, with %d components" % (self.logitsShape, dim))
        if self.teacherEntries < 0:
            raise ValueError("negative number of entries")
        most = torch.finfo(torch.float32).max                    # (log2(e) / T and T^2 are taken in fp32)
        if not 0.0 <= self.alpha <= 1.0 or not 1.45 / most < self.temperature < most ** 0.5:
            raise ValueError("alpha in [0, 1] and a positive temperature with 1.45 / T and T^2 in fp32's range expected")
        self.samples = self.logitsShape[0] // dim
        self.teacherShape, self.lossShape, self.statsShape = (self.samples, self.teacherEntries), (self.samples,), (3, self.samples)
        self._calls = {}

    def getLogitsShape(self): return self.logitsShape
    def getClasses(self): return MULTIVECTOR_DIM[self.algebra] * self.logitsShape[1]
    def getTeacherShape(self): return self.teacherShape
    def getLossShape(self): return self.lossShape
    def getStatsShape(self): return self.statsShape
    def getAlgebra(self): return self.algebra

    def _call(self, dtype):
        call = self._calls.get(dtype)
        if call is None:
            d = _lib.DistillDesc()
            d.dtype, d.algebra, d.batch, d.units = _DTYPES[dtype], _ALGEBRAS[self.algebra], self.samples, self.logitsShape[1]
            d.entries, d.alpha, d.temperature = self.teacherEntries, self.alpha, self.temperature
            sample, stats = (torch.float32, self.lossShape), (torch.float32, self.statsShape)
            operands = [("logits", dtype, self.logitsShape), ("labels", torch.int64, self.lossShape), ("teacherLogits", dtype, self.teacherShape),
                        ("teacherIndices", torch.int64, self.teacherShape)]
            call = self._calls[dtype] = (_Entry("pcb_distill_fwd", d, operands + [("loss",) + sample, ("stats",) + stats]),
                                         _Entry("pcb_distill_bwd", d, operands + [("stats",) + stats, ("gradLoss",) + sample, ("gradLogits", dtype, self.logitsShape)]))
        return call


def _teacher(descriptor, teacher, index):
    if descriptor.teacherEntries == 0:
        return None, None
    if teacher is None or index is None:
        raise ValueError("the descriptor has %d entries of a teacher" % descriptor.teacherEntries)
    return teacher, index


def distillFwd(logitsTensor, labels, teacherLogits, teacherIndices, lossTensor, statsTensor, descriptor):
    """Losses (fp32, one per sample) of logits against ``labels`` (int64, None: no such term; a value outside the classes leaves a sample's out) and
    the teacher's logits at ``teacherIndices`` (int64; an index outside the classes leaves an entry out). ``statsTensor`` (fp32,
    ``getStatsShape()``) is kept for ``distillBwd`` and may be None."""
    _input_device(logitsTensor, "logits")
    teacher, index = _teacher(descriptor, teacherLogits, teacherIndices)
    if lossTensor is None:
        raise ValueError("loss expected")
    fwd, operands = descriptor._call(logitsTensor.dtype)[0], (logitsTensor, labels, teacher, index, lossTensor, statsTensor)
    if descriptor.samples:
        fwd.call(None, 0, *operands)
    else:
        fwd.check(*operands)


def distillBwd(logitsTensor, labels, teacherLogits, teacherIndices, statsTensor, gradLoss, gradLogits, descriptor):
    """The gradient of the logits, ``gradLoss`` (fp32) being that of each sample's loss. ``gradLogits`` must not be the logits themselves."""
    _input_device(logitsTensor, "logits")
    teacher, index = _teacher(descriptor, teacherLogits, teacherIndices)
    if statsTensor is None or gradLoss is None or gradLogits is None:
        raise ValueError("stats, gradLoss and gradLogits expected")
    bwd, operands = descriptor._call(logitsTensor.dtype)[1], (logitsTensor, labels, teacher, index, statsTensor, gradLoss, gradLogits)
    if descriptor.samples:
        bwd.call(None, 0, *operands)
    else:
        bwd.check(*operands)
