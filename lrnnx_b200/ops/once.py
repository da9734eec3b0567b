"""Gradients without gradients of their own, and which calls need the autograd function at all."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def _dual_level():
    """Whether tensors may carry forward-mode tangents now (the level is torch's own; a torch that does not tell has them asked)."""
    return getattr(forward_ad, "_current_level", 0) >= 0


def recorded(*tensors):
    """Whether a call on these (None is passed over) goes through its autograd function: one of them requires a gradient, or carries a
    forward-mode tangent, which the function refuses and a bare launch would drop."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return _dual_level() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _OnceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, count, *tensors):
        return tensors[count:]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("lrnnx_b200: the gradient of this operator cannot be differentiated again")


def once(inputs, grads):
    """``grads`` of a backward pass; where it runs with ``create_graph``, tied to the ``inputs`` they were formed from, so that
    to differentiate them again is an error and not silently a constant; so is an upstream gradient with a forward-mode tangent."""
    if not torch.is_grad_enabled() and not _dual_level():
        return grads
    at = [i for i, t in enumerate(grads) if t is not None]
    tied = _OnceFn.apply(len(inputs), *inputs, *[grads[i] for i in at])
    grads = list(grads)
    for i, t in zip(at, tied):
        grads[i] = t
    return tuple(grads)
