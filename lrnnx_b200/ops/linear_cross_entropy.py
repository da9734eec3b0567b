"""Next-token cross entropy of a language model's head without its logits (``b200_lce_fwd / bwd``).

``linear_cross_entropy(hidden, weight, labels)`` is ``cross_entropy(hidden @ weight.T, labels)``
with the product, the log-sum-exp and, in the backward, softmax minus one-hot in one pass over
tensor-core tiles: of the (rows, classes) logits nothing is kept but one float32 log-sum-exp a row,
and the backward forms their gradient in pieces of the vocabulary (at most 1 GiB at a time).  lrnnx's
LM returns logits and has no loss (lrnnx/architectures/language_model.py:615-727); with 50280
classes the logits of 16384 tokens are the largest tensor of a training step.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .mamba_block import _DT, _stream

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _rows(t):
    """t with its last dimension contiguous and rows that do not overlap."""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1) and t.stride(0) >= t.shape[-1] else t.contiguous()


def _work(a, name, like):
    a.work_bytes = getattr(_lib.lib(), name)(ctypes.byref(a))
    work = torch.empty(max(a.work_bytes, 1), dtype=torch.uint8, device=like.device)
    a.work = work.data_ptr()
    return work


class LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction):
        ctx.shapes = hidden.shape, weight.shape
        labels_shape = labels.shape
        hidden, weight = _rows(hidden.reshape(-1, hidden.shape[-1])), _rows(weight)
        labels = labels.reshape(-1).to(torch.int64).contiguous()
        a = _lib.struct("b200_lce_args")()
        a.rows, a.features = hidden.shape
        a.classes, a.ignore_index, a.reduction = weight.shape[0], ignore_index, reduction
        a.dtype = _lib.enum(_DT[hidden.dtype])
        with _lib.on_device(hidden):
            lse = torch.empty(a.rows, dtype=torch.float32, device=hidden.device)
            loss = torch.empty(labels_shape if reduction == 0 else (), dtype=torch.float32, device=hidden.device)
            count = torch.empty((), dtype=torch.float32, device=hidden.device)
            a.hidden, a.weight, a.labels = hidden.data_ptr(), weight.data_ptr(), labels.data_ptr()
            a.hidden_rs, a.weight_rs = hidden.stride(0), weight.stride(0)
            a.lse, a.loss, a.count = lse.data_ptr(), loss.data_ptr(), count.data_ptr()
            work = _work(a, "b200_lce_fwd_work_bytes", hidden)
            _lib.call("b200_lce_fwd", a, _stream(hidden))
            del work
        ctx.save_for_backward(hidden, weight, labels, lse, count)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    def backward(ctx, grad):
        hidden, weight, labels, lse, count = ctx.saved_tensors
        need_h, need_w = ctx.needs_input_grad[:2]
        a = _lib.struct("b200_lce_args")()
        a.rows, a.features = hidden.shape
        a.classes, a.ignore_index, a.reduction = weight.shape[0], ctx.ignore_index, ctx.reduction
        a.dtype = _lib.enum(_DT[hidden.dtype])
        with _lib.on_device(hidden):
            grad = grad.to(torch.float32).contiguous()
            dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if need_h else None
            dw = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if need_w else None
            a.hidden, a.weight, a.labels = hidden.data_ptr(), weight.data_ptr(), labels.data_ptr()
            a.hidden_rs, a.weight_rs = hidden.stride(0), weight.stride(0)
            a.lse, a.count, a.dloss = lse.data_ptr(), count.data_ptr(), grad.data_ptr()
            if need_h:
                a.dhidden, a.dhidden_rs = dh.data_ptr(), dh.stride(0)
            if need_w:
                a.dweight, a.dweight_rs = dw.data_ptr(), dw.stride(0)
            work = _work(a, "b200_lce_bwd_work_bytes", hidden)
            _lib.call("b200_lce_bwd", a, _stream(hidden))
            del work
        return dh.view(ctx.shapes[0]) if need_h else None, dw, None, None, None


def linear_cross_entropy(hidden, weight, labels, ignore_index=-100, reduction="mean"):
    """``cross_entropy(hidden @ weight.T, labels)`` with a float32 result: the mean over the labels
    that are not ``ignore_index`` (zero where there are none), their sum, or with ``reduction="none"``
    the loss of every row, zero for ignored ones.  hidden (..., features) and weight (classes,
    features) float32, float16 or bfloat16 alike; labels (...) integer.  A label outside [0, classes)
    has no loss and no gradient, as in ``cross_entropy``.  Gradients for hidden and weight."""
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
    return LinearCrossEntropyFn.apply(hidden, weight, labels, ignore_index, _REDUCTIONS[reduction])
