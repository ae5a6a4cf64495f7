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
from .descriptors import MULTIVECTOR_DIM, Algebra, FilterLayout
from .ops import _ALGEBRAS, _DTYPES, Device, _check_tensor, _dense_desc, _OnDevice, _ptr, _stream

BLOCK = 128


class Filter8:
    """A dense filter held in 8 bits: ``[D, I, O]`` (``FilterLayout.IO``) or ``[D, O, I]`` (``FilterLayout.OI``), without the leading axis for
    real-valued layers. Filled by ``quantizeFilter8``; one object serves ``dense8Fwd`` and ``dense8Bwd``.

    ``values`` is a view of the e4m3 numbers (its rows start on 16 bytes), ``scales`` the bytes e + 127 of the blocks,
    ``[D, blocks of rows, blocks of columns]``. Numbers of another origin can be copied into both."""

    def __init__(self, filterShape, algebra=Algebra.QUATERNION, filterLayout=FilterLayout.IO, device="cuda"):
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
        pitch = (cols + 15) // 16 * 16
        self._storage = torch.zeros((dim, rows, pitch), dtype=torch.uint8, device=device)
        self.values = self._storage.view(torch.float8_e4m3fn)[:, :, :cols].reshape(self.shape) if pitch == cols else \
            self._storage.view(torch.float8_e4m3fn)[:, :, :cols]
        if self.values.dim() != len(self.shape):
            self.values = self.values[0]
        self.scales = torch.full((dim, (rows + BLOCK - 1) // BLOCK, (cols + BLOCK - 1) // BLOCK), 127, dtype=torch.uint8, device=device)

    @property
    def device(self):
        return self._storage.device

    def dequantize(self):
        """The fp32 values that the filter stands for."""
        dim, (rows, cols) = self._storage.shape[0], self.shape[-2:]
        scale = (self.scales.int() << 23).view(torch.float32)
        scale = scale.repeat_interleave(BLOCK, 1)[:, :rows].repeat_interleave(BLOCK, 2)[:, :, :cols]
        return (self.values.reshape(dim, rows, cols).float() * scale).reshape(self.shape)


def _check_filter8(filter8, descriptor, device):
    if not isinstance(filter8, Filter8):
        raise ValueError("filter must be a Filter8 (see quantizeFilter8)")
    if filter8.shape != tuple(descriptor.getFilterShape()) or filter8.algebra != descriptor.getAlgebra() or filter8.filterLayout != descriptor.getFilterLayout():
        raise ValueError("filter mismatch: %s vs expected %s" % (filter8.shape, tuple(descriptor.getFilterShape())))
    if filter8.device != device:
        raise ValueError("filter is on %s, the input on %s" % (filter8.device, device))


def _check_input(t, name, shape):
    if t.dtype not in _DTYPES:
        raise ValueError("%s dtype %s: float32, float16 or bfloat16 expected" % (name, t.dtype))
    _check_tensor(t, name, shape=shape)


def quantizeFilter8(filterTensor, filter8):
    """Rounds a filter of 16- or 32-bit numbers into ``filter8``."""
    _check_input(filterTensor, "filter", filter8.shape)
    if filter8.device != filterTensor.device:
        raise ValueError("the Filter8 is on %s, the filter on %s" % (filter8.device, filterTensor.device))
    d = _lib.DenseDesc()
    oi = filter8.filterLayout == FilterLayout.OI
    d.dtype, d.algebra, d.filter_oi = _DTYPES[filterTensor.dtype], _ALGEBRAS[filter8.algebra], int(oi)
    d.in_features, d.out_features = filter8.shape[-1 if oi else -2], filter8.shape[-2 if oi else -1]
    dev = Device.get(filterTensor.device)
    with _OnDevice(dev.index):
        _lib.check(_lib.lib().pcb_quantize_filter8(ctypes.byref(d), _ptr(filterTensor), _ptr(filter8._storage), _ptr(filter8.scales), _stream()))


def dense8Fwd(inputTensor, filter8, biasTensor, outputTensor, descriptor, context=None, engine=_lib.ENGINE_AUTO):
    """``denseFwd`` with a filter held in 8 bits and the input quantised along its features. Input, bias and output share a type."""
    dev = Device.get(inputTensor.device)
    context = context or dev.getContext()
    _check_input(inputTensor, "input", descriptor.getInputShape())
    _check_filter8(filter8, descriptor, inputTensor.device)
    _check_tensor(outputTensor, "output", inputTensor.dtype, descriptor.getOutputShape())
    if biasTensor is not None:
        if not descriptor.isBiasUsed():
            raise ValueError("Bias application is not configured for this scalar Dense operation")
        _check_tensor(biasTensor, "bias", inputTensor.dtype, descriptor.getBiasShape())
    if inputTensor.numel() == 0:
        return
    d = _dense_desc(descriptor, inputTensor.dtype, context, engine, has_bias=biasTensor is not None)
    L = _lib.lib()
    with dev.accessControl, _OnDevice(dev.index):
        need = getattr(d, "_fwd8_need", None)
        if need is None:
            need = d._fwd8_need = L.pcb_qdense8_fwd_workspace_size(ctypes.byref(d))
        ws = dev.requestWorkspace(need)
        _lib.check(L.pcb_qdense8_fwd(ctypes.byref(d), _ptr(inputTensor), _ptr(filter8._storage), _ptr(filter8.scales), _ptr(biasTensor),
                                     _ptr(outputTensor), _ptr(ws), ws.numel(), _stream()))
        dev._after_op()


def dense8Bwd(inputTensor, filter8, gradTensor, filterGradTensor, inputGradTensor, descriptor, context=None, engine=_lib.ENGINE_AUTO):
    """``denseBwd`` in 8 bits: the filter gradient (input-major, ``[D, I, O]``, whatever the filter layout) from the input and the output
    gradient quantised along the samples, the input gradient from the filter and the output gradient quantised along the features."""
    dev = Device.get(inputTensor.device)
    context = context or dev.getContext()
    _check_input(inputTensor, "input", descriptor.getInputShape())
    _check_filter8(filter8, descriptor, inputTensor.device)
    _check_tensor(gradTensor, "grad", inputTensor.dtype, descriptor.getOutputShape())
    _check_tensor(filterGradTensor, "filterGrad", inputTensor.dtype)
    i, o = descriptor.getInputChannels(), descriptor.getOutputChannels()
    if tuple(filterGradTensor.shape) != filter8.shape[:-2] + (i, o):
        raise ValueError("filterGrad shape mismatch: %s vs expected %s" % (tuple(filterGradTensor.shape), filter8.shape[:-2] + (i, o)))
    need_dx = descriptor.isInputGradientRequired()
    if need_dx:
        _check_tensor(inputGradTensor, "inputGrad", inputTensor.dtype, descriptor.getInputShape())
    if inputTensor.numel() == 0:
        filterGradTensor.zero_()
        return
    d = _dense_desc(descriptor, inputTensor.dtype, context, engine, require_input_grad=need_dx)
    L = _lib.lib()
    with dev.accessControl, _OnDevice(dev.index):
        need = getattr(d, "_bwd8_need", None)
        if need is None:
            need = d._bwd8_need = L.pcb_qdense8_bwd_workspace_size(ctypes.byref(d))
        ws = dev.requestWorkspace(need)
        _lib.check(L.pcb_qdense8_bwd(ctypes.byref(d), _ptr(inputTensor), _ptr(filter8._storage), _ptr(filter8.scales), _ptr(gradTensor),
                                     _ptr(filterGradTensor), _ptr(inputGradTensor) if need_dx else None, _ptr(ws), ws.numel(), _stream()))
        dev._after_op()
