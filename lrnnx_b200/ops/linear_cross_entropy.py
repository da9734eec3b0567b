"""Next-token cross entropy of a language model's head without its logits (``b200_lce_fwd / bwd``).

``linear_cross_entropy(hidden, weight, labels)`` is ``cross_entropy(hidden @ weight.T, labels)``
with the product, the log-sum-exp and, in the backward, softmax minus one-hot in one pass over
tensor-core tiles: of the (rows, classes) logits nothing is kept but one float32 log-sum-exp a row,
and the backward forms their gradient in pieces of the vocabulary (at most 1 GiB at a time).  lrnnx's
LM returns logits and has no loss (lrnnx/architectures/language_model.py:615-727); with 50280
classes the logits of 16384 tokens are the largest tensor of a training step.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .mamba_block import _DT
from .once import once, recorded

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _rows(t):
    """t with its last dimension contiguous and rows that do not overlap."""
    if (t.stride(-1) == 1 or t.shape[-1] == 1) and t.stride(0) >= t.shape[-1]:
        return t
    return t.clone(memory_format=torch.contiguous_format) if t.shape[0] == 1 else t.contiguous()      # a single row of any pitch counts as contiguous


@functools.lru_cache(maxsize=None)
def _setup():
    return _lib.packer("b200_lce_args"), {t: _lib.enum(n) for t, n in _DT.items()}


def _call(name, hidden, weight, labels, ignore_index, reduction, lse, loss, count, dloss, dh, dw):
    pack, codes = _setup()
    rows, features = hidden.shape
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    head = (rows, ignore_index, weight.shape[0], features, codes[hidden.dtype], reduction, hidden.data_ptr(), weight.data_ptr(), labels.data_ptr(),
            hidden.stride(0), weight.stride(0), lse.data_ptr(), at(loss), at(count), at(dloss), at(dh), at(dw), features, features)
    work_bytes = getattr(_lib.lib(), name + "_work_bytes")(pack(*head, 0, 0))
    work = torch.empty(max(work_bytes, 1), dtype=torch.uint8, device=hidden.device)
    _lib.call(name, pack(*head, work.data_ptr(), work_bytes), _lib.stream_of(hidden))


def _forward(hidden, weight, labels, ignore_index, reduction, shape):
    with _lib.on_device(hidden):
        lse = torch.empty(hidden.shape[0], dtype=torch.float32, device=hidden.device)
        loss = torch.empty(shape if reduction == 0 else (), dtype=torch.float32, device=hidden.device)
        count = torch.empty((), dtype=torch.float32, device=hidden.device) if reduction == 1 else None
        _call("b200_lce_fwd", hidden, weight, labels, ignore_index, reduction, lse, loss, count, None, None, None)
    return loss, lse, count


class LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction):
        ctx.shape = hidden.shape
        hidden = _rows(hidden.reshape(-1, hidden.shape[-1]))
        weight = _rows(weight)
        flat = labels.reshape(-1).to(torch.int64).contiguous()
        loss, lse, count = _forward(hidden, weight, flat, ignore_index, reduction, labels.shape)
        ctx.save_for_backward(hidden, weight, flat, lse, count)
        ctx.meta = ignore_index, reduction
        return loss

    @staticmethod
    def backward(ctx, grad):
        hidden, weight, labels, lse, count = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        with _lib.on_device(hidden):
            given, grad = grad, grad.to(torch.float32).contiguous()
            dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if need_h else None
            dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if need_w else None
            _call("b200_lce_bwd", hidden, weight, labels, *ctx.meta, lse, None, count, grad, dh, dw)
        return *once((hidden, weight, given), (dh.view(ctx.shape) if need_h else None, dw)), None, None, None


def linear_cross_entropy(hidden, weight, labels, ignore_index=-100, reduction="mean"):
    """``cross_entropy(hidden @ weight.T, labels)`` with a float32 result: the mean over the labels
    that are not ``ignore_index`` (zero where there are none), their sum, or with ``reduction="none"``
    the loss of every row, zero for ignored ones.  hidden (..., features) and weight (classes,
    features) float32, float16 or bfloat16 alike; labels (...) integer.  A label outside [0, classes)
    has no loss and no gradient, as in ``cross_entropy``; a row without a target may hold anything.
    float32 operands are multiplied as sums of three bfloat16, so that an infinite one gives NaN (also where
    a product with it is infinite): classes are not masked by weights of -inf.  Gradients for hidden and
    weight; forward-mode derivatives are an error."""
    if reduction not in _REDUCTIONS:
        raise RuntimeError(f"linear_cross_entropy: reduction must be one of {', '.join(_REDUCTIONS)}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or labels.shape != hidden.shape[:-1]:
        raise RuntimeError("linear_cross_entropy: hidden (..., features), weight (classes, features) and labels (...) expected")
    if hidden.dtype not in _DT or weight.dtype != hidden.dtype or not hidden.is_cuda:
        raise RuntimeError("linear_cross_entropy: hidden and weight must be float32 / float16 / bfloat16 CUDA tensors of one dtype")
    if weight.device != hidden.device or labels.device != hidden.device:
        raise RuntimeError("linear_cross_entropy: hidden, weight and labels must be on one device")
    if labels.is_floating_point() or labels.is_complex() or labels.dtype == torch.bool:
        raise RuntimeError("linear_cross_entropy: labels must be integers")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise RuntimeError("linear_cross_entropy: there must be classes and features")
    if labels.numel() == 0:                        # no rows: a sum over nothing, with gradients of zero
        zero = (hidden.sum() + weight[:0].sum()).float()
        return zero.expand(labels.shape) if reduction == "none" else zero
    # copies that the kernels need are made here, where autograd sees them: what is saved is then what came in, which second derivatives go by
    hidden, weight = _rows(hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])), _rows(weight)
    if recorded(hidden, weight):
        return LinearCrossEntropyFn.apply(hidden, weight, labels, ignore_index, _REDUCTIONS[reduction])
    return _forward(hidden, weight, labels.reshape(-1).to(torch.int64).contiguous(), ignore_index, _REDUCTIONS[reduction], labels.shape)[0]
