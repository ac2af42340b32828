"""A layer's input kept in 8 bits for its backward pass.

Training a layer stack on a whole graph is bound by what autograd keeps: every linear map holds
its ``n x F`` input in full until the weight gradient is formed (model/GCN.py:14-16,
model/SGC.py:14).  ``save_int8`` keeps it as one byte per element and one byte per group of 32
features, and the weight gradient is formed from those bytes (``SavedInt8.weight_grad``).  An
activation ``x if x > 0 else slope * x`` in front of the map is folded in: the sign of a code is
the sign of ``x``, so the activation keeps nothing of its own (``SavedInt8.input_grad``).

``linear_saved_int8`` is the layer built of these; ``nn.GCNConv`` and ``nn.SGConv`` use it with
``checkpoint="int8"``.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from ._lib import TYPES, element_type


def checked_slope(slope):
    """``slope`` as the kernels hold it; what they cannot hold is refused."""
    slope = float(slope)
    if not (math.isfinite(slope) and slope >= 0.0):
        raise ValueError(f"the activation's slope must be finite and not negative, got {slope}")
    # what the kernels compute with; a slope that 32 bits cannot hold is refused, not turned into another one
    held = ctypes.c_float(slope).value
    if math.isinf(held) or (held == 0.0) != (slope == 0.0) or (held == 1.0) != (slope == 1.0):
        raise ValueError(f"the activation's slope is not a 32-bit number: {slope}")
    return held


def activated(x, slope):
    """``x if x > 0 else slope * x`` by torch's operators."""
    if slope == 1.0:
        return x
    return torch.relu(x) if slope == 0.0 else torch.nn.functional.leaky_relu(x, slope)


def unit_rows(t):
    """``t`` with unit stride along its rows and rows that do not overlap (a copy if need be)."""
    n, f = t.shape
    if (f > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < f):
        return t.contiguous()
    return t


def _ld(t):
    return max(t.stride(0), t.shape[1])


class SavedInt8:
    """An ``n x F`` activation in 8 bits: ``codes`` int8 ``[n, 32 * ceil(F / 32)]``, ``steps``
    uint8 ``[n, ceil(F / 32)]`` (the group's exponent plus 127), ``slope`` and the ``dtype`` it
    came from."""

    def __init__(self, codes, steps, shape, slope, dtype):
        self.codes, self.steps, self.shape = codes, steps, tuple(shape)
        self.slope, self.dtype = checked_slope(slope), dtype
        n, F = self.shape
        groups = -(-F // _lib.SAVED8_GROUP)
        for name, t, kind, width in (("codes", codes, torch.int8, groups * _lib.SAVED8_GROUP),
                                     ("steps", steps, torch.uint8, groups)):
            if t.dtype != kind or tuple(t.shape) != (n, width) or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"{name} must be a contiguous {kind} tensor of shape {(n, width)} on the GPU")
        if steps.device != codes.device:
            raise ValueError("codes and steps are on different devices")
        if codes.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")
        if dtype not in TYPES:
            raise TypeError(f"saved activations are float32 or bfloat16, got {dtype}")

    @classmethod
    def _of(cls, codes, steps, shape, slope, dtype):
        """The same of parts that were just made to fit."""
        saved = object.__new__(cls)
        saved.codes, saved.steps, saved.shape, saved.slope, saved.dtype = codes, steps, shape, slope, dtype
        return saved

    @property
    def nbytes(self):
        return self.codes.numel() + self.steps.numel()

    @property
    def device(self):
        return self.codes.device

    def restore(self, dtype=None):
        """The values the codes stand for, ``n x F`` (exact in either type)."""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in TYPES:
            raise TypeError(f"saved activations are restored as float32 or bfloat16, not {dtype}")
        n, F = self.shape
        out = torch.empty(n, F, dtype=dtype, device=self.device)
        _lib.call_on(self.device, _lib.load().sgnn_restore8, TYPES[dtype], n, F, self.codes.data_ptr(),
                     self.steps.data_ptr(), self.slope, out.data_ptr(), F)
        return out

    def _grad(self, grad, width, what):
        element_type(grad, what)
        if grad.dim() != 2 or grad.shape[0] != self.shape[0] or (width is not None and grad.shape[1] != width):
            raise ValueError(f"{what} must have shape ({self.shape[0]}, {'H' if width is None else width}), "
                             f"got {tuple(grad.shape)}")
        if grad.device != self.device:
            raise ValueError(f"{what} is on {grad.device}, the saved activation on {self.device}")
        return unit_rows(grad.detach())

    def weight_grad(self, grad):
        """``grad.T @ values``: the gradient ``[H, F]`` of a weight applied to the activation, from
        the gradient ``[n, H]`` of its output, in ``grad``'s type."""
        grad = self._grad(grad, None, "the output's gradient")
        (n, F), H = self.shape, grad.shape[1]
        if n == 0 or H == 0:
            return torch.zeros(H, F, dtype=grad.dtype, device=self.device)
        lib = _lib.load()
        dW = torch.empty(H, F, dtype=grad.dtype, device=self.device)
        nbytes = lib.sgnn_saved8_weight_grad_workspace_bytes(n, F, H)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        _lib.call_on(self.device, lib.sgnn_saved8_weight_grad, TYPES[grad.dtype], n, F, H, self.codes.data_ptr(),
                     self.steps.data_ptr(), self.slope, grad.data_ptr(), _ld(grad), dW.data_ptr(), F, ws.data_ptr(),
                     nbytes)
        return dW

    def input_grad(self, grad):
        """``grad * act'(x)``: the gradient of the activation's input from that of its output, a
        tensor of its own."""
        given, grad = grad, self._grad(grad, self.shape[1], "the activation's gradient")
        if self.slope == 1.0:
            return grad.clone() if grad.data_ptr() == given.data_ptr() else grad
        n, F = self.shape
        out = torch.empty(n, F, dtype=grad.dtype, device=self.device)
        _lib.call_on(self.device, _lib.load().sgnn_saved8_input_grad, TYPES[grad.dtype], n, F, self.codes.data_ptr(),
                     self.slope, grad.data_ptr(), _ld(grad), out.data_ptr(), F)
        return out


def _empty(n, F, device):
    groups = -(-F // _lib.SAVED8_GROUP)
    return (torch.empty(n, groups * _lib.SAVED8_GROUP, dtype=torch.int8, device=device),
            torch.empty(n, groups, dtype=torch.uint8, device=device))


def save_int8(x, slope=1.0):
    """``x if x > 0 else slope * x`` in 8 bits (``slope`` 1: no activation, 0: ReLU).  A part of a backward
    pass of one's own: neither it nor what is made of it is differentiable."""
    code = element_type(x, "the activation")
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"the activation must be a matrix with at least one column, got {tuple(x.shape)}")
    slope = checked_slope(slope)
    x = unit_rows(x.detach())
    n, F = x.shape
    codes, steps = _empty(n, F, x.device)
    _lib.call_on(x.device, _lib.load().sgnn_save8, code, n, F, x.data_ptr(), _ld(x), slope, codes.data_ptr(),
                 steps.data_ptr())
    return SavedInt8._of(codes, steps, (n, F), slope, x.dtype)


def _linear(x, weight, slope, codes=None, steps=None):
    x, w = unit_rows(x.detach()), unit_rows(weight.detach())
    (n, F), H = x.shape, w.shape[0]
    y = torch.empty(n, H, dtype=x.dtype, device=x.device)
    _lib.call_on(x.device, _lib.load().sgnn_saved8_linear, TYPES[x.dtype], n, F, H, x.data_ptr(), _ld(x), w.data_ptr(),
                 _ld(w), slope, None if codes is None else codes.data_ptr(), None if steps is None else steps.data_ptr(),
                 y.data_ptr(), H)
    return y


class _LinearSaved(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, slope):
        codes, steps = _empty(*x.shape, x.device)
        ctx.save_for_backward(codes, steps, weight)
        ctx.meta = (tuple(x.shape), slope, x.dtype)
        return _linear(x, weight, slope, codes, steps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        codes, steps, weight = ctx.saved_tensors
        (n, F), slope, dtype = ctx.meta
        dx = dw = None
        grad = unit_rows(grad)
        if ctx.needs_input_grad[0]:
            w, H = unit_rows(weight), weight.shape[0]
            dx = torch.empty(n, F, dtype=dtype, device=grad.device)
            _lib.call_on(grad.device, _lib.load().sgnn_saved8_linear_grad, TYPES[dtype], n, F, H, codes.data_ptr(), slope,
                         grad.data_ptr(), _ld(grad), w.data_ptr(), _ld(w), dx.data_ptr(), F)
        if ctx.needs_input_grad[1]:
            dw = SavedInt8._of(codes, steps, (n, F), slope, dtype).weight_grad(grad)
        return dx, dw, None


def linear_saved_int8(x, weight, slope=1.0):
    """``act(x) @ weight.T`` with ``act(x) = x if x > 0 else slope * x``, keeping nothing of its
    input but the 8-bit codes for the backward pass.  The output and ``x``'s gradient are those of
    the full activation; the weight's gradient is formed from the codes (off by half a step of
    their group at most, element by element).  An infinite or NaN element makes its row's outputs
    NaN (in bfloat16 an infinity may stay one).  Neither forward-mode nor second derivatives: autograd refuses both."""
    code = element_type(x, "the input")
    if element_type(weight, "the weight") != code:
        raise TypeError(f"the input is {x.dtype}, the weight {weight.dtype}")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"need an (n, F) input and an (H, F) weight, got {tuple(x.shape)} and {tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError(f"the input is on {x.device}, the weight on {weight.device}")
    slope = checked_slope(slope)
    # an operand with a forward-mode tangent, too: autograd refuses it there, here it would be lost
    if (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad)
            or any(unpack_dual(t).tangent is not None for t in (x, weight))):
        return _LinearSaved.apply(x, weight, slope)
    return _linear(x, weight, slope)
