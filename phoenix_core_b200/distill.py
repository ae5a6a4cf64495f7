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
from .ops import _ALGEBRAS, _DTYPES, Device, _check_tensor, _OnDevice, _ptr, _stream


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
        if not 0.0 <= self.alpha <= 1.0 or not 0.0 < self.temperature < float("inf"):
            raise ValueError("alpha in [0, 1] and a positive temperature expected")
        self.samples = self.logitsShape[0] // dim
        self._desc = {}

    def getLogitsShape(self): return self.logitsShape
    def getClasses(self): return MULTIVECTOR_DIM[self.algebra] * self.logitsShape[1]
    def getTeacherShape(self): return (self.samples, self.teacherEntries)
    def getLossShape(self): return (self.samples,)
    def getStatsShape(self): return (3, self.samples)
    def getAlgebra(self): return self.algebra

    def _c(self, dtype):
        d = self._desc.get(dtype)
        if d is None:
            d = _lib.DistillDesc()
            d.dtype, d.algebra, d.batch, d.units = _DTYPES[dtype], _ALGEBRAS[self.algebra], self.samples, self.logitsShape[1]
            d.entries, d.alpha, d.temperature = self.teacherEntries, self.alpha, self.temperature
            self._desc[dtype] = d
        return d


def _check(t, name, like, dtype, shape):
    _check_tensor(t, name, dtype, shape)
    if t.device != like.device:
        raise ValueError("%s is on %s, the logits on %s" % (name, t.device, like.device))


def _check_operands(logits, labels, teacher, index, descriptor):
    if logits.dtype not in _DTYPES:
        raise ValueError("logits dtype %s: float32, float16 or bfloat16 expected" % logits.dtype)
    _check_tensor(logits, "logits", shape=descriptor.getLogitsShape())
    if labels is not None:
        _check(labels, "labels", logits, torch.int64, descriptor.getLossShape())
    if descriptor.teacherEntries > 0:
        if teacher is None or index is None:
            raise ValueError("the descriptor has %d entries of a teacher" % descriptor.teacherEntries)
        _check(teacher, "teacherLogits", logits, logits.dtype, descriptor.getTeacherShape())
        _check(index, "teacherIndices", logits, torch.int64, descriptor.getTeacherShape())


def distillFwd(logitsTensor, labels, teacherLogits, teacherIndices, lossTensor, statsTensor, descriptor):
    """Losses (fp32, one per sample) of logits against ``labels`` (int64, None: no such term; a value outside the classes leaves a sample's out) and
    the teacher's logits at ``teacherIndices`` (int64; an index outside the classes leaves an entry out). ``statsTensor`` (fp32,
    ``getStatsShape()``) is kept for ``distillBwd`` and may be None."""
    x = logitsTensor
    _check_operands(x, labels, teacherLogits, teacherIndices, descriptor)
    _check(lossTensor, "loss", x, torch.float32, descriptor.getLossShape())
    if statsTensor is not None:
        _check(statsTensor, "stats", x, torch.float32, descriptor.getStatsShape())
    if x.numel() == 0:
        return
    teacher = descriptor.teacherEntries > 0
    dev = Device.get(x.device)
    with _OnDevice(dev.index):
        _lib.check(_lib.lib().pcb_distill_fwd(ctypes.byref(descriptor._c(x.dtype)), _ptr(x), _ptr(labels), _ptr(teacherLogits) if teacher else None,
                                              _ptr(teacherIndices) if teacher else None, _ptr(lossTensor), _ptr(statsTensor), _stream()))


def distillBwd(logitsTensor, labels, teacherLogits, teacherIndices, statsTensor, gradLoss, gradLogits, descriptor):
    """The gradient of the logits, ``gradLoss`` (fp32) being that of each sample's loss. ``gradLogits`` must not be the logits themselves."""
    x = logitsTensor
    _check_operands(x, labels, teacherLogits, teacherIndices, descriptor)
    _check(statsTensor, "stats", x, torch.float32, descriptor.getStatsShape())
    _check(gradLoss, "gradLoss", x, torch.float32, descriptor.getLossShape())
    _check(gradLogits, "gradLogits", x, x.dtype, descriptor.getLogitsShape())
    if x.numel() == 0:
        return
    teacher = descriptor.teacherEntries > 0
    dev = Device.get(x.device)
    with _OnDevice(dev.index):
        _lib.check(_lib.lib().pcb_distill_bwd(ctypes.byref(descriptor._c(x.dtype)), _ptr(x), _ptr(labels), _ptr(teacherLogits) if teacher else None,
                                              _ptr(teacherIndices) if teacher else None, _ptr(statsTensor), _ptr(gradLoss), _ptr(gradLogits), _stream()))
