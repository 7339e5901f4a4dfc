"""Rows of logits with a label each, as the operators over them take them:
argument checks and the layout their C entries are given.

Logits are [V], [T, V] or [B, S, V] (more leading dimensions are flattened), of
float32, bfloat16 or float16, with any strides between rows: a next-token view
``logits[:, :-1]`` is read where it lies.  A tensor whose last dimension is not
dense is copied.  Labels have the logits' leading shape and are int64.
"""

import torch
from torch.autograd.forward_ad import unpack_dual

from framework import capi

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def check(logits, labels, *others):
    """The checks every operator makes: devices, types, shapes."""
    capi.require(logits.is_cuda and labels.is_cuda, "logits, labels must be GPU tensors")
    capi.require(logits.dtype in DTYPES, "logits must be float32, bfloat16 or float16")
    capi.require(labels.dtype == torch.int64, "labels must be int64")
    capi.require(logits.dim() >= 1 and logits.size(-1) >= 1 and
                 labels.shape == logits.shape[:-1],
                 "logits must be [..., V] with V >= 1 and labels of their leading shape")
    device = logits.get_device()
    capi.require(labels.get_device() == device, "labels must be on the GPU of the logits")
    for name, t in others:
        if t is not None:
            capi.require(t.is_cuda and t.get_device() == device,
                         f"{name} must be a tensor on the GPU of the logits")


def differentiated(logits):
    """Whether a call goes through its autograd function: where logits need a
    gradient, and where they carry a tangent, which is refused there."""
    return (logits.requires_grad and torch.is_grad_enabled() or
            unpack_dual(logits).tangent is not None)


class _Once(torch.autograd.Function):
    """A gradient of the logits that refuses to be differentiated."""

    @staticmethod
    def forward(ctx, dlogits, _):
        return dlogits.view_as(dlogits)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("operators over rows of logits have no second derivatives")


def once(dlogits):
    """A backward's answer, which autograd takes for a constant.  Where a graph of the
    gradients is made (create_graph) it refuses a second derivative instead, also
    where the gradient that came in needs none: dlogits depends on the logits."""
    if not torch.is_grad_enabled():
        return dlogits
    return _Once.apply(dlogits, dlogits.new_empty(0).requires_grad_(True))


def layout(logits):
    """(logits, B, S, V, batch stride, row stride), copied only if it must be."""
    V, d = logits.size(-1), logits.dim()
    if d > 3 or (V > 1 and logits.stride(-1) != 1):
        logits = logits.contiguous()
    if d == 3:
        B, S = logits.size(0), logits.size(1)
        return logits, B, S, V, logits.stride(0), logits.stride(1)
    if d == 2:
        return logits, 1, logits.size(0), V, 0, logits.stride(0)
    return logits, 1, logits.numel() // V, V, 0, V


def saved(logits, labels, kept, per_row):
    """``layout`` of the logits that a backward gets back, with labels and ``kept``,
    of ``per_row`` numbers a row, dense.  It is that of the tensor given: what a
    saved-tensor hook put elsewhere comes back as a copy with strides of its own."""
    rows, n = layout(logits), labels.numel()
    capi.require(0 <= logits.get_device() == labels.get_device() == kept.get_device() and
                 rows[1] * rows[2] == n and kept.numel() == per_row * n,
                 "autograd gave back other tensors than were saved")
    return labels.contiguous(), kept.contiguous(), *rows


def per_token(t, name, shape):
    """A float32 tensor that broadcasts to `shape`, dense."""
    capi.require(t.dtype == torch.float32, f"{name} must be float32")
    if t.shape != shape:
        try:
            t = t.expand(shape)
        except RuntimeError:
            raise RuntimeError(f"{name} must broadcast to the labels' shape {tuple(shape)}, "
                               f"got {tuple(t.shape)}") from None
    return t.contiguous()
