"""Embedding lookup with a scale, and its gradient by sorted tokens (``b200_embed_fwd / bwd``).

``token_embedding(ids, weight)`` takes the place of nn.Embedding in the language model
(lrnnx/architectures/language_model.py:198-240).  Its gradient adds the rows of each token in float32 in
the order of their positions, so it is the same at every call, and rounds once.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .mamba_block import _DT, _stream


def _args(ids, features, classes, dtype, scale, padding_idx):
    a = _lib.struct("b200_embed_args")()
    a.tokens, a.features, a.classes = ids.numel(), features, classes
    a.dtype, a.ids_wide = _lib.enum(_DT[dtype]), int(ids.dtype == torch.int64)
    a.scale, a.padding_idx = scale, padding_idx
    a.ids = ids.data_ptr()
    return a


class TokenEmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        if weight.stride(1) != 1 or weight.stride(0) < weight.shape[1]:
            weight = weight.contiguous()
        flat = ids.reshape(-1).contiguous()
        classes, features = weight.shape
        with _lib.on_device(weight):
            out = torch.empty(*ids.shape, features, dtype=weight.dtype, device=weight.device)
            a = _args(flat, features, classes, weight.dtype, scale, padding_idx)
            a.weight, a.out = weight.data_ptr(), out.data_ptr()
            a.weight_rs, a.out_rs = weight.stride(0), features
            _lib.call("b200_embed_fwd", a, _stream(weight))
        ctx.save_for_backward(flat)
        ctx.meta = classes, scale, padding_idx
        return out

    @staticmethod
    def backward(ctx, dout):
        flat, = ctx.saved_tensors
        classes, scale, padding_idx = ctx.meta
        features = dout.shape[-1]
        dout = dout.reshape(-1, features)
        if dout.stride(1) != 1 and features > 1:
            dout = dout.contiguous()
        with _lib.on_device(dout):
            dweight = torch.empty(classes, features, dtype=dout.dtype, device=dout.device)
            a = _args(flat, features, classes, dout.dtype, scale, padding_idx)
            a.dout, a.dweight = dout.data_ptr(), dweight.data_ptr()
            a.dout_rs, a.dweight_rs = dout.stride(0), features
            a.work_bytes = _lib.lib().b200_embed_bwd_work_bytes(ctypes.byref(a))
            work = torch.empty(max(a.work_bytes, 1), dtype=torch.uint8, device=dout.device)
            a.work = work.data_ptr()
            _lib.call("b200_embed_bwd", a, _stream(dout))
            del work
        return None, dweight, None, None


def token_embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: ids (...) int32 or int64, weight (classes, features) float32, float16 or
    bfloat16 -> (..., features).  The gradient of row ``padding_idx`` is zero.  An id outside
    [0, classes) reads nothing: its row is NaN, and it adds to no gradient."""
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise RuntimeError("token_embedding: weight (classes, features) expected")
    if weight.dtype not in _DT or not weight.is_cuda:
        raise RuntimeError("token_embedding: weight must be a float32 / float16 / bfloat16 CUDA tensor")
    if ids.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("token_embedding: ids must be int32 or int64")
    if ids.device != weight.device:
        raise RuntimeError("token_embedding: ids and weight must be on one device")
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise RuntimeError("token_embedding: padding_idx must be a row of weight")
        padding_idx %= weight.shape[0]
    if ids.numel() == 0:
        return weight[:0].sum() + torch.empty(*ids.shape, weight.shape[1], dtype=weight.dtype, device=weight.device)
    return TokenEmbeddingFn.apply(ids, weight, float(scale), -1 if padding_idx is None else padding_idx)
