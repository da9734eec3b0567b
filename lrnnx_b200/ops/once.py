"""Gradients without gradients of their own."""
from __future__ import annotations

import torch


class _OnceFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, count, *tensors):
        return tensors[count:]

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("lrnnx_b200: the gradient of this operator cannot be differentiated again")


def once(inputs, grads):
    """``grads`` of a backward pass; where it runs with ``create_graph``, tied to the ``inputs`` they were formed from, so that
    to differentiate them again is an error and not silently a constant."""
    if not torch.is_grad_enabled():
        return grads
    at = [i for i, t in enumerate(grads) if t is not None]
    tied = _OnceFn.apply(len(inputs), *inputs, *[grads[i] for i in at])
    grads = list(grads)
    for i, t in zip(at, tied):
        grads[i] = t
    return tuple(grads)
