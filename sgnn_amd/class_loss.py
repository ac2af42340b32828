"""Cross-entropy of a label head of any width, without keeping its logits.

The label head of the reference forms ``embedding @ Wt``, its softmax and its gradient as full
``rows x classes`` matrices (model/SGNN.py:397-399).  ``class_cross_entropy`` runs over the classes
in pieces, forward and backward, so what it needs grows with the rows plus the classes and not
with their product.
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import element_type
from .saved8 import unit_rows


def _weight_layout(w):
    """``w`` (V x D) with unit stride along one of its directions, and its strides."""
    V, D = w.shape
    sv, sd = w.stride()
    if D == 1 or V == 1:                             # a stride of a direction of length 1 says nothing
        w = w.contiguous()
        return w, D, 1
    if not ((sd == 1 and sv >= D) or (sv == 1 and sd >= V)):
        w = w.contiguous()
        sv, sd = w.stride()
    return w, sv, sd


class _ClassXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, labels, idx, mean, all_rows=False):
        x, (w, sv, sd) = unit_rows(x.detach()), _weight_layout(weight.detach())
        (B, D), V, dev = x.shape, w.shape[0], x.device
        lib, dtype = _lib.load(), _lib.TYPES[x.dtype] | (_lib.ALL_ROWS if all_rows else 0)
        kept = torch.empty(4 * B + 1, dtype=torch.float32, device=dev)   # statistics, 1 / counted rows, row losses
        out = torch.empty(() if mean else (B,), dtype=torch.float32, device=dev)
        nbytes = lib.sgnn_class_xent_workspace_bytes(dtype, B, D, V, 0)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        at = kept.data_ptr()
        rows, loss, share = (at + 12 * B + 4, out.data_ptr(), at + 12 * B) if mean else (out.data_ptr(), None, None)
        _lib.call_on(dev, lib.sgnn_class_xent_forward, dtype, B, D, V, x.data_ptr(), max(x.stride(0), D), w.data_ptr(),
                     sv, sd, labels.data_ptr(), labels.numel(), None if idx is None else idx.data_ptr(), at, rows, loss,
                     share, ws.data_ptr(), nbytes)
        ctx.save_for_backward(x, w, labels, idx, kept)
        ctx.layout = (sv, sd, mean, dtype)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, w, labels, idx, kept = ctx.saved_tensors
        (B, D), V, dev = x.shape, w.shape[0], x.device
        sv, sd, mean, dtype = ctx.layout
        lib = _lib.load()
        grad = grad.contiguous()
        dx = torch.empty(B, D, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw, dsv, dsd = None, D, 1
        if ctx.needs_input_grad[1]:                  # in the weight's own layout
            if sd == 1:
                dw = torch.empty(V, D, dtype=w.dtype, device=dev)
            else:
                dw, dsv, dsd = torch.empty(D, V, dtype=w.dtype, device=dev).t(), 1, V
        nbytes = lib.sgnn_class_xent_workspace_bytes(dtype, B, D, V, 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        at = kept.data_ptr()
        _lib.call_on(dev, lib.sgnn_class_xent_backward, dtype, B, D, V, x.data_ptr(), max(x.stride(0), D), w.data_ptr(),
                     sv, sd, labels.data_ptr(), labels.numel(), None if idx is None else idx.data_ptr(), at,
                     grad.data_ptr(), at + 12 * B if mean else None, None if dx is None else dx.data_ptr(), D,
                     None if dw is None else dw.data_ptr(), dsv, dsd, ws.data_ptr(), nbytes)
        return dx, dw, None, None, None, None


def _ids(t, what, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int64 or t.dim() != 1:
        raise TypeError(f"{what} must be a 1-D int64 tensor")
    if t.device != device:
        raise ValueError(f"{what} are on {t.device}, x on {device}")
    return t.contiguous()


def class_cross_entropy(x, weight, labels, idx=None, reduction="mean"):
    """Cross-entropy of ``x @ weight.T`` (``x`` B x D, ``weight`` V x D, both float32 or both
    bfloat16) against ``labels[idx]`` (``labels`` if ``idx`` is None; int64), in float32.

    A row whose index or label is out of range (-1, say) has no class: its loss and its part of
    either gradient are 0.  ``reduction="mean"`` is the mean over the other rows (0 if there are
    none), ``"none"`` the loss of each row.  ``weight`` may be a transposed view (``Wt.t()``); its
    gradient comes in the same layout.  An infinite or NaN element makes the losses it takes part
    in NaN or infinite; in bfloat16 a class whose logit is -infinity has p = 0 instead."""
    if reduction not in ("mean", "none"):
        raise ValueError(f"reduction must be 'mean' or 'none', got {reduction!r}")
    if element_type(x, "x") != element_type(weight, "the weight"):
        raise TypeError(f"x is {x.dtype}, the weight {weight.dtype}")
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1] or x.shape[1] == 0 or weight.shape[0] == 0:
        raise ValueError(f"need (B, D) rows and a (V, D) weight, got {tuple(x.shape)} and {tuple(weight.shape)}")
    if weight.device != x.device:
        raise ValueError(f"x is on {x.device}, the weight on {weight.device}")
    labels = _ids(labels, "labels", x.device)
    if idx is not None:
        idx = _ids(idx, "idx", x.device)
    rows = labels.numel() if idx is None else idx.numel()
    if rows != x.shape[0]:
        raise ValueError(f"{x.shape[0]} rows but {rows} {'labels' if idx is None else 'indices'}")
    if x.shape[0] == 0:                              # nothing counts: 0, with zero gradients
        nothing = x.float().sum(1) + weight[:0].float().sum()
        return nothing.sum() if reduction == "mean" else nothing
    if labels.numel() == 0:
        raise ValueError("labels are empty")
    return _ClassXent.apply(x, weight, labels, idx, reduction == "mean")
