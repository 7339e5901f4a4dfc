"""What the differentiable operators share of autograd's corners: gradients of
first order, in reverse, and nothing else.

A tangent (forward mode) is refused by the operator's autograd function, which
is therefore entered wherever an input carries one; a second derivative is
refused where somebody goes on to take it.
"""

import torch
from torch.autograd import forward_ad


def differentiated(*tensors):
    """Whether a call goes through its autograd function: where an input needs a
    gradient, and where one carries a tangent, which is refused there."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if getattr(forward_ad, "_current_level", 0) < 0:    # no tangents anywhere
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _Once(torch.autograd.Function):
    """A gradient that refuses to be differentiated."""

    @staticmethod
    def forward(ctx, what, grad, _):
        ctx.what = what
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"{ctx.what} has no second derivatives")


def once(what, *grads):
    """A backward's answers, which autograd takes for constants.  Where a graph of the
    gradients is made (create_graph) they refuse a second derivative instead, also
    where the gradient that came in needs none: they depend on the inputs."""
    if not torch.is_grad_enabled():
        return grads
    return tuple(g if g is None else _Once.apply(what, g, g.new_empty(0).requires_grad_(True))
                 for g in grads)
