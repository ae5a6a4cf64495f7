"""The dense layer in 8-bit floating point: ``quantizeFilter8``, ``dense8Fwd`` and ``dense8Bwd`` beside ``denseFwd`` /
``denseBwd`` (no counterpart in the reference, whose layers are 16- and 32-bit).

A block of values is held as e4m3 numbers times 2^e, e the smallest whole number with max|x| <= 448 * 2^e (0 for a block of
zeros, -126 at least). Filters have one scale for each 128 x 128 block of every component and are kept in that form
(``Filter8``); activations and output gradients come in 16 or 32 bits and are quantised inside the call, with one scale for each
128 values along the axis that the product sums over: features for the output and the input gradient, samples for the filter
gradient. Products are exact, sums are held in 32 bits, and each result is rounded once to its type. Infinities and NaN become NaN.

Descriptors, layouts, streams, workspaces and errors are those of ``denseFwd`` / ``denseBwd``; every algebra is taken.
"""
import ctypes

import torch

from . import _lib
from .context import Context
from .descriptors import MULTIVECTOR_DIM, Algebra, FilterLayout
from .ops import _ALGEBRAS, _DTYPES, Device, _build_dense_desc, _Entry, _input_device

BLOCK = 128


class Filter8:
    """A dense filter held in 8 bits: ``[D, I, O]`` (``FilterLayout.IO``) or ``[D, O, I]`` (``FilterLayout.OI``), without the leading axis for
    real-valued layers. Filled by ``quantizeFilter8``; one object serves ``dense8Fwd`` and ``dense8Bwd``.

    ``values`` is a view of the e4m3 numbers (its rows start on 16 bytes), ``scales`` the bytes e + 127 of the blocks,
    ``[D, blocks of rows, blocks of columns]``. Numbers of another origin can be copied into both. ``fill=False`` leaves them unset, for a filter that is
    rounded into the object next (a zero filter otherwise)."""

    def __init__(self, filterShape, algebra=Algebra.QUATERNION, filterLayout=FilterLayout.IO, device="cuda", fill=True):
        self.shape = tuple(int(s) for s in filterShape)
        self.algebra, self.filterLayout = algebra, filterLayout
        dim = MULTIVECTOR_DIM[algebra]
        if filterLayout not in (FilterLayout.IO, FilterLayout.OI):
            raise ValueError("a dense filter has the layout IO or OI")
        if len(self.shape) not in ((2, 3) if algebra == Algebra.REAL else (3,)) or (len(self.shape) == 3 and self.shape[0] != dim):
            raise ValueError("filter shape mismatch: %s for %d components" % (self.shape, dim))
        rows, cols = self.shape[-2:]
        if rows <= 0 or cols <= 0:
            raise ValueError("invalid filter shape %s" % (self.shape,))
        storage, blocks = Filter8.shapes(self.shape, algebra)
        self._storage = (torch.zeros if fill else torch.empty)(storage, dtype=torch.uint8, device=device)
        self.scales = torch.full(blocks, 127, dtype=torch.uint8, device=device) if fill else torch.empty(blocks, dtype=torch.uint8, device=device)
        self._entries = {}

    @staticmethod
    def shapes(filterShape, algebra):
        """Shapes of the bytes that hold a filter's numbers and its scales."""
        rows, cols = filterShape[-2:]
        dim = MULTIVECTOR_DIM[algebra]
        return (dim, rows, (cols + 15) // 16 * 16), (dim, (rows + BLOCK - 1) // BLOCK, (cols + BLOCK - 1) // BLOCK)

    @property
    def values(self):
        v = self._storage.view(torch.float8_e4m3fn)[:, :, :self.shape[-1]]
        return v if len(self.shape) == 3 else v[0]

    @property
    def device(self):
        return self._storage.device

    def dequantize(self):
        """The fp32 values that the filter stands for."""
        dim, (rows, cols) = self._storage.shape[0], self.shape[-2:]
        scale = (self.scales.int() << 23).view(torch.float32)
        scale = scale.repeat_interleave(BLOCK, 1)[:, :rows].repeat_interleave(BLOCK, 2)[:, :, :cols]
        return (self.values.reshape(dim, rows, cols).float() * scale).reshape(self.shape)


class _Call:
    """What a call with a descriptor needs and does not change."""

    def __init__(self, descriptor, dtype, engine, flag, forward):
        context = Context({})                                # (the formulation that a context chooses has no meaning here)
        desc = _build_dense_desc(descriptor, dtype, context, engine, has_bias=forward and flag, require_input_grad=not forward and flag)
        L = _lib.lib()
        self.workspace = (L.pcb_qdense8_fwd_workspace_size if forward else L.pcb_qdense8_bwd_workspace_size)(ctypes.byref(desc))
        shape, out, self.filter = descriptor.getInputShape(), descriptor.getOutputShape(), tuple(descriptor.getFilterShape())
        self.algebra, self.layout, self.empty = descriptor.getAlgebra(), descriptor.getFilterLayout(), shape[0] == 0
        held = Filter8.shapes(self.filter, self.algebra)
        operands = [("input", dtype, shape), ("filter", torch.uint8, held[0]), ("filter scales", torch.uint8, held[1])]
        if forward:
            operands += [("bias", dtype, descriptor.getBiasShape()), ("output", dtype, out)]
        else:
            grad = self.filter[:-2] + (descriptor.getInputChannels(), descriptor.getOutputChannels())
            operands += [("grad", dtype, out), ("filterGrad", dtype, grad), ("inputGrad", dtype, shape)]
        self.entry = _Entry("pcb_qdense8_fwd" if forward else "pcb_qdense8_bwd", desc, operands)

    @staticmethod
    def of(descriptor, dtype, engine, flag, forward):
        cache = descriptor.__dict__.setdefault("_pcb_dense8", {})
        key = (dtype, engine, flag, forward)
        call = cache.get(key)
        if call is None:
            call = cache[key] = _Call(descriptor, dtype, engine, flag, forward)
        return call

    def check_filter(self, filter8):
        if not isinstance(filter8, Filter8):
            raise ValueError("filter must be a Filter8 (see quantizeFilter8)")
        if filter8.shape != self.filter or filter8.algebra != self.algebra or filter8.filterLayout != self.layout:
            raise ValueError("filter mismatch: %s vs expected %s" % (filter8.shape, self.filter))


def quantizeFilter8(filterTensor, filter8):
    """Rounds a filter of 16- or 32-bit numbers into ``filter8``."""
    _input_device(filterTensor, "filter")
    entry = filter8._entries.get(filterTensor.dtype)
    if entry is None:
        d = _lib.DenseDesc()
        oi = filter8.filterLayout == FilterLayout.OI
        d.dtype, d.algebra, d.filter_oi = _DTYPES[filterTensor.dtype], _ALGEBRAS[filter8.algebra], int(oi)
        d.in_features, d.out_features = filter8.shape[-1 if oi else -2], filter8.shape[-2 if oi else -1]
        held = Filter8.shapes(filter8.shape, filter8.algebra)
        entry = filter8._entries[filterTensor.dtype] = _Entry("pcb_quantize_filter8", d, [
            ("filter", filterTensor.dtype, filter8.shape), ("8-bit filter", torch.uint8, held[0]), ("8-bit filter's scales", torch.uint8, held[1])])
    entry.call(None, 0, filterTensor, filter8._storage, filter8.scales)


def dense8Fwd(inputTensor, filter8, biasTensor, outputTensor, descriptor, context=None, engine=_lib.ENGINE_AUTO):
    """``denseFwd`` with a filter held in 8 bits and the input quantised along its features. Input, bias and output share a type."""
    index, bias = _input_device(inputTensor, "input"), biasTensor is not None
    call = _Call.of(descriptor, inputTensor.dtype, engine, bias, True)
    call.check_filter(filter8)
    if bias and not descriptor.isBiasUsed():
        raise ValueError("Bias application is not configured for this scalar Dense operation")
    if outputTensor is None:
        raise ValueError("output expected")
    if call.empty:
        return call.entry.check(inputTensor, filter8._storage, filter8.scales, biasTensor, outputTensor)
    dev = Device.at(index)
    with dev.accessControl:
        ws = dev.requestWorkspace(call.workspace)
        call.entry.call(ws, 0, inputTensor, filter8._storage, filter8.scales, biasTensor, outputTensor)
        dev._after_op()


def dense8Bwd(inputTensor, filter8, gradTensor, filterGradTensor, inputGradTensor, descriptor, context=None, engine=_lib.ENGINE_AUTO):
    """``denseBwd`` in 8 bits: the filter gradient (input-major, ``[D, I, O]``, whatever the filter layout) from the input and the output
    gradient quantised along the samples, the input gradient from the filter and the output gradient quantised along the features."""
    index, need_dx = _input_device(inputTensor, "input"), descriptor.isInputGradientRequired()
    call = _Call.of(descriptor, inputTensor.dtype, engine, need_dx, False)
    call.check_filter(filter8)
    if gradTensor is None or filterGradTensor is None or (need_dx and inputGradTensor is None):
        raise ValueError("grad, filterGrad and, where the descriptor asks for it, inputGrad expected")
    operands = (inputTensor, filter8._storage, filter8.scales, gradTensor, filterGradTensor, inputGradTensor if need_dx else None)
    if call.empty:
        call.entry.check(*operands)
        filterGradTensor.zero_()
        return
    dev = Device.at(index)
    with dev.accessControl:
        ws = dev.requestWorkspace(call.workspace)
        call.entry.call(ws, 0, *operands)
        dev._after_op()
