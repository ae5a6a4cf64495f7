"""PyTorch autograd front end of the engine: ``QConv2dFunction`` / ``QDenseFunction`` and two small modules.

The reference is driven from a framework plugin (its TensorFlow ops call ``upstride::conv2DFwd`` / ``conv2DBwd`` /
``denseFwd`` / ``denseBwd`` of ``src/upstride.hpp:18-86`` from the op's compute callback). This module is the same
thing for PyTorch: each function's ``forward`` calls the forward entry point, its ``backward`` the backward entry
point, on the caller's tensors and the current CUDA stream. Tensors use the engine's layouts: activations
``[D*N, C, H, W]`` (or ``[D*N, H, W, C]``) with the multivector components stacked on the batch axis, filters
``[D, Co, Ci, kh, kw]`` (OIHW) and friends, dense filters ``[D, I, O]`` / ``[D, O, I]``, bias ``[D, C]``.

The engine's backward pass has no bias gradient (the framework side owns the bias in the reference too): it is the
sum of the output gradient over batch and pixels per component and channel, computed here with one torch reduction.
"""
import torch

from . import _lib
from .descriptors import (Algebra, Conv2DBwdDescriptor, Conv2DFwdDescriptor, DataFormat, DenseBwdDescriptor, DenseFwdDescriptor,
                          FilterLayout, MULTIVECTOR_DIM, Padding)
from .dense8 import Filter8, dense8Bwd, dense8Fwd, quantizeFilter8
from .distill import DistillDescriptor, distillBwd, distillFwd
from .ops import conv2DBwd, conv2DFwd, denseBwd, denseFwd
from .residual_norm import ResidualNormDescriptor, residualNormBwd, residualNormFwd


class QConv2dFunction(torch.autograd.Function):
    """``y = QConv2dFunction.apply(x, w, bias, stride, dilation, padding, explicit_pad, groups, algebra, data_format,
    filter_layout, real_valued_input, context)``.

    padding: a ``Padding`` value; ``explicit_pad`` = (top, left, bottom, right) when it is ``Padding.EXPLICIT``.
    ``real_valued_input``: x is a real ``[N, C, H, W]`` tensor entering a hyper-complex layer (no input gradient
    exists then, reference ``src/conv2d.hpp:384-396``)."""

    @staticmethod
    def forward(ctx, x, w, bias, stride=1, dilation=1, padding=Padding.VALID, explicit_pad=(), groups=1,
                algebra=Algebra.QUATERNION, data_format=DataFormat.NCHW, filter_layout=FilterLayout.OIHW,
                real_valued_input=False, context=None):
        x, w = x.contiguous(), w.contiguous()
        args = (tuple(x.shape), tuple(w.shape), stride, dilation, padding, tuple(explicit_pad), groups, algebra, data_format, filter_layout)
        fwd = Conv2DFwdDescriptor(*args, bias is not None, real_valued_input)
        y = torch.empty(fwd.getOutputShape(), dtype=x.dtype, device=x.device)
        conv2DFwd(x, w, None if bias is None else bias.contiguous(), y, fwd, context)
        ctx.save_for_backward(x, w)
        ctx.args, ctx.real, ctx.context, ctx.has_bias = args, real_valued_input, context, bias is not None
        ctx.channel_axis = 1 if data_format == DataFormat.NCHW else 3
        ctx.dim = MULTIVECTOR_DIM[algebra]
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dy = dy.contiguous()
        need_dx = ctx.needs_input_grad[0] and not ctx.real
        bwd = Conv2DBwdDescriptor(*ctx.args, need_dx, ctx.real)
        dw = torch.empty_like(w)
        dx = torch.empty_like(x) if need_dx else None
        conv2DBwd(x, w, dy, dw, dx, bwd, ctx.context)
        db = None
        if ctx.has_bias and ctx.needs_input_grad[2]:
            g = dy.view(ctx.dim, -1, *dy.shape[1:])
            axes = [a for a in range(g.dim()) if a not in (0, ctx.channel_axis + 1)]
            db = g.float().sum(dim=axes).to(dy.dtype)
        return (dx, dw, db) + (None,) * 10


class QDenseFunction(torch.autograd.Function):
    """``y = QDenseFunction.apply(x, w, bias, algebra, filter_layout, context)`` with x ``[D*B, I]`` and w ``[D, I, O]``
    (``FilterLayout.IO``) or ``[D, O, I]`` (``FilterLayout.OI``). The engine always emits the filter gradient as
    ``[D, I, O]`` (reference ``src/backend/cudnn/dense.hpp:187-195``); it is transposed back here for OI filters so
    that the gradient has the shape of the parameter."""

    @staticmethod
    def forward(ctx, x, w, bias, algebra=Algebra.QUATERNION, filter_layout=FilterLayout.IO, context=None):
        x, w = x.contiguous(), w.contiguous()
        fwd = DenseFwdDescriptor(tuple(x.shape), tuple(w.shape), algebra, filter_layout, bias is not None)
        y = torch.empty(fwd.getOutputShape(), dtype=x.dtype, device=x.device)
        denseFwd(x, w, None if bias is None else bias.contiguous(), y, fwd, context)
        ctx.save_for_backward(x, w)
        ctx.algebra, ctx.layout, ctx.context, ctx.has_bias = algebra, filter_layout, context, bias is not None
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dy = dy.contiguous()
        need_dx = ctx.needs_input_grad[0]
        bwd = DenseBwdDescriptor(tuple(x.shape), tuple(w.shape), ctx.algebra, ctx.layout, need_dx)
        i, o = bwd.getInputChannels(), bwd.getOutputChannels()
        dw_io = torch.empty(w.shape[:-2] + (i, o), dtype=w.dtype, device=w.device)
        dx = torch.empty_like(x) if need_dx else None
        denseBwd(x, w, dy, dw_io, dx, bwd, ctx.context)
        dw = dw_io if ctx.layout == FilterLayout.IO else dw_io.transpose(-1, -2).contiguous()
        db = None
        if ctx.has_bias and ctx.needs_input_grad[2]:
            dim = MULTIVECTOR_DIM[ctx.algebra]
            db = dy.view(dim, -1, dy.shape[1]).float().sum(1).to(dy.dtype)
        return dx, dw, db, None, None, None


class QDense8Function(torch.autograd.Function):
    """``y = QDense8Function.apply(x, w, bias, algebra, filter_layout)``: ``QDenseFunction`` in 8 bits. The filter is rounded for the call; forward and
    backward use the same rounded filter, and its gradient is given to the filter as it was before."""

    @staticmethod
    def forward(ctx, x, w, bias, algebra=Algebra.QUATERNION, filter_layout=FilterLayout.IO):
        x, w = x.contiguous(), w.contiguous()
        fwd = DenseFwdDescriptor(tuple(x.shape), tuple(w.shape), algebra, filter_layout, bias is not None)
        filter8 = Filter8(tuple(w.shape), algebra, filter_layout, x.device, fill=False)
        quantizeFilter8(w, filter8)
        y = torch.empty(fwd.getOutputShape(), dtype=x.dtype, device=x.device)
        dense8Fwd(x, filter8, None if bias is None else bias.contiguous(), y, fwd)
        ctx.save_for_backward(x)
        ctx.filter8, ctx.has_bias = filter8, bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        (x,) = ctx.saved_tensors
        dy, f = dy.contiguous(), ctx.filter8
        need_dx = ctx.needs_input_grad[0]
        bwd = DenseBwdDescriptor(tuple(x.shape), f.shape, f.algebra, f.filterLayout, need_dx)
        dw = torch.empty(f.shape[:-2] + (bwd.getInputChannels(), bwd.getOutputChannels()), dtype=x.dtype, device=x.device)
        dx = torch.empty_like(x) if need_dx else None
        dense8Bwd(x, f, dy, dw, dx, bwd)
        if f.filterLayout == FilterLayout.OI:
            dw = dw.transpose(-1, -2).contiguous()
        db = None
        if ctx.has_bias and ctx.needs_input_grad[2]:
            dim = MULTIVECTOR_DIM[f.algebra]
            db = dy.view(dim, -1, dy.shape[1]).float().sum(1).to(dy.dtype)
            db = db if dim > 1 else db[0]
        return dx, dw, db, None, None


class ResidualNormFunction(torch.autograd.Function):
    """``y, h = ResidualNormFunction.apply(residual, branch, gate, post_weight, pre_weight, algebra, residual_scale, epsilon)`` (see
    ``residualNormFwd``). ``branch`` None: ``y`` is the residual itself. Weights (fp32) and gate may be None."""

    @staticmethod
    def forward(ctx, residual, branch, gate, post, pre, algebra=Algebra.REAL, residual_scale=1.0, epsilon=1e-6):
        dim = MULTIVECTOR_DIM[algebra]
        residual = residual.contiguous()
        branch, gate, post, pre = (None if t is None else t.contiguous() for t in (branch, gate, post, pre))
        d = ResidualNormDescriptor(tuple(residual.shape), 0 if gate is None else gate.shape[0] // dim, algebra, residual_scale, epsilon)
        y = None if branch is None else torch.empty_like(residual)
        h = torch.empty_like(residual)
        stats = torch.empty(d.getStatsShape(), dtype=torch.float32, device=residual.device)
        residualNormFwd(residual, branch, gate, post, pre, y, h, stats, d)
        ctx.save_for_backward(residual if y is None else y, branch, gate, post, pre, stats)
        ctx.descriptor = d
        ctx.set_materialize_grads(False)
        return (residual if y is None else y), h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        y, branch, gate, post, pre, stats = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 8
        dy, dh = (None if t is None else t.contiguous() for t in (dy, dh))
        need = ctx.needs_input_grad
        dx = torch.empty_like(y)
        db = None if branch is None else torch.empty_like(branch)
        dgate = torch.empty_like(gate) if gate is not None and need[2] else None
        dpost = torch.empty_like(post) if post is not None and need[3] else None
        dpre = torch.empty_like(pre) if pre is not None and need[4] else None
        if dh is None:                                     # nothing came back through the norm behind the block
            residualNormBwd(y, branch, gate, post, None, stats, dy, None, dx, db, dgate, dpost, None, ctx.descriptor)
            if dpre is not None:
                dpre.zero_()
        else:
            residualNormBwd(y, branch, gate, post, pre, stats, dy, dh, dx, db, dgate, dpost, dpre, ctx.descriptor)
        return dx, db, dgate, dpost, dpre, None, None, None


class DistillFunction(torch.autograd.Function):
    """``losses = DistillFunction.apply(logits, labels, teacher_logits, teacher_indices, alpha, temperature, algebra)`` (see ``distillFwd``): one
    fp32 loss per sample. Gradients go to the logits alone."""

    @staticmethod
    def forward(ctx, logits, labels, teacher_logits, teacher_indices, alpha=0.5, temperature=1.0, algebra=Algebra.QUATERNION):
        logits = logits.contiguous()
        entries = 0 if teacher_indices is None else teacher_indices.shape[1]
        labels, teacher_logits, teacher_indices = (None if t is None else t.contiguous() for t in (labels, teacher_logits, teacher_indices))
        d = DistillDescriptor(tuple(logits.shape), entries, alpha, temperature, algebra)
        losses = torch.empty(d.getLossShape(), dtype=torch.float32, device=logits.device)
        stats = torch.empty(d.getStatsShape(), dtype=torch.float32, device=logits.device)
        distillFwd(logits, labels, teacher_logits, teacher_indices, losses, stats, d)
        ctx.save_for_backward(logits, labels, teacher_logits, teacher_indices, stats)
        ctx.descriptor = d
        return losses

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        logits, labels, teacher_logits, teacher_indices, stats = ctx.saved_tensors
        dlogits = torch.empty_like(logits)
        distillBwd(logits, labels, teacher_logits, teacher_indices, stats, grad.contiguous(), dlogits, ctx.descriptor)
        return (dlogits,) + (None,) * 6


class QConv2d(torch.nn.Module):
    """Quaternion (or other algebra) convolution layer with He-normal filters over the D*Ci*kh*kw real inputs."""

    def __init__(self, in_channels, out_channels, kernel_size, stride=1, padding=Padding.SAME, dilation=1, groups=1, bias=True,
                 algebra=Algebra.QUATERNION, dtype=torch.float16, device="cuda", context=None):
        super().__init__()
        d = MULTIVECTOR_DIM[algebra]
        kh, kw = (kernel_size, kernel_size) if isinstance(kernel_size, int) else kernel_size
        std = (2.0 / (d * (in_channels // groups) * kh * kw)) ** 0.5
        self.weight = torch.nn.Parameter(torch.randn((d, out_channels, in_channels // groups, kh, kw), device=device) .mul_(std).to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros((d, out_channels), dtype=dtype, device=device)) if bias else None
        self.stride, self.padding, self.dilation, self.groups, self.algebra, self.context = stride, padding, dilation, groups, algebra, context

    def forward(self, x):
        return QConv2dFunction.apply(x, self.weight, self.bias, self.stride, self.dilation, self.padding, (), self.groups, self.algebra,
                                     DataFormat.NCHW, FilterLayout.OIHW, False, self.context)


class QDense(torch.nn.Module):
    def __init__(self, in_features, out_features, bias=True, algebra=Algebra.QUATERNION, dtype=torch.float16, device="cuda", context=None):
        super().__init__()
        d = MULTIVECTOR_DIM[algebra]
        self.weight = torch.nn.Parameter(torch.randn((d, in_features, out_features), device=device).mul_((2.0 / (d * in_features)) ** 0.5).to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros((d, out_features), dtype=dtype, device=device)) if bias else None
        self.algebra, self.context = algebra, context

    def forward(self, x):
        return QDenseFunction.apply(x, self.weight, self.bias, self.algebra, FilterLayout.IO, self.context)


class QDense8(QDense):
    """``QDense`` computed in 8 bits: the filter stays in `dtype` and is rounded in every call, as training needs it. ``pack`` rounds it once, for calls
    without gradients from then on, until ``unpack`` (or the next call with gradients); a filter that changes meanwhile has to be packed again."""

    def __init__(self, in_features, out_features, bias=True, algebra=Algebra.QUATERNION, dtype=torch.bfloat16, device="cuda"):
        super().__init__(in_features, out_features, bias, algebra, dtype, device)
        if algebra == Algebra.REAL:
            self.weight = torch.nn.Parameter(self.weight.detach()[0].clone())
            self.bias = torch.nn.Parameter(self.bias.detach()[0].clone()) if bias else None
        self.filter8 = None

    def pack(self):
        if self.filter8 is None:
            self.filter8 = Filter8(tuple(self.weight.shape), self.algebra, FilterLayout.IO, self.weight.device)
        quantizeFilter8(self.weight.detach().contiguous(), self.filter8)
        return self

    def unpack(self):
        self.filter8 = None
        return self

    def forward(self, x):
        if self.filter8 is None or torch.is_grad_enabled():
            self.filter8 = None
            return QDense8Function.apply(x, self.weight, self.bias, self.algebra, FilterLayout.IO)
        x = x.contiguous()
        fwd = DenseFwdDescriptor(tuple(x.shape), self.filter8.shape, self.algebra, FilterLayout.IO, self.bias is not None)
        y = torch.empty(fwd.getOutputShape(), dtype=x.dtype, device=x.device)
        dense8Fwd(x, self.filter8, self.bias, y, fwd)
        return y


class QResidualNorm(torch.nn.Module):
    """The norms behind and before a block: ``y, h = layer(residual, branch, gate)`` with y the residual path's next value and h what the next block reads;
    ``branch`` None in front of the first block."""

    def __init__(self, features, algebra=Algebra.QUATERNION, residual_scale=1.0, epsilon=1e-6, device="cuda"):
        super().__init__()
        self.post_weight = torch.nn.Parameter(torch.ones(features, dtype=torch.float32, device=device))
        self.pre_weight = torch.nn.Parameter(torch.ones(features, dtype=torch.float32, device=device))
        self.algebra, self.residual_scale, self.epsilon = algebra, residual_scale, epsilon

    def forward(self, residual, branch=None, gate=None):
        return ResidualNormFunction.apply(residual, branch, gate, None if branch is None else self.post_weight, self.pre_weight, self.algebra,
                                          self.residual_scale, self.epsilon)


__all__ = ["QConv2dFunction", "QDenseFunction", "QConv2d", "QDense", "QDense8Function", "ResidualNormFunction", "DistillFunction", "QDense8", "QResidualNorm"]
