"""Embedding lookup with a scale, and its gradient by sorted tokens (``b200_embed_fwd / bwd``).

``token_embedding(ids, weight)`` takes the place of nn.Embedding in the language model
(lrnnx/architectures/language_model.py:198-511).  Its gradient adds the rows of each token in float32 in
an order that the list of ids fixes (partial sums of up to 16 neighbours in the sorted list, then eight interleaved shares of those), so it
is the same at every call, and rounds once; other ids in the list can change a row's last bits.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .mamba_block import _DT
from .once import once, recorded


@functools.lru_cache(maxsize=None)
def _setup():
    return _lib.packer("b200_embed_args"), {t: _lib.enum(n) for t, n in _DT.items()}


def _lookup(ids, weight, classes, features, scale, padding_idx):
    """out, and the ids in a row"""
    if weight.stride(1) != 1 or weight.stride(0) < features:
        weight = weight.contiguous()
    flat = ids if ids.is_contiguous() else ids.contiguous()
    pack, codes = _setup()
    dtype = weight.dtype
    with _lib.on_device(weight):
        out = weight.new_empty(ids.shape + (features,))
        _lib.call("b200_embed_fwd", pack(flat.numel(), padding_idx, classes, features, codes[dtype], flat.dtype == torch.int64, scale, 0,
                                         flat.data_ptr(), weight.data_ptr(), 0, out.data_ptr(), 0, weight.stride(0), features, 0, 0, 0, 0),
                  _lib.stream_of(weight))
    return out, flat


class TokenEmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        out, flat = _lookup(ids, weight, *weight.shape, scale, padding_idx)
        ctx.save_for_backward(flat)
        ctx.meta = weight.shape[0], scale, padding_idx
        return out

    @staticmethod
    def backward(ctx, dout):
        flat, = ctx.saved_tensors
        classes, scale, padding_idx = ctx.meta
        features = dout.shape[-1]
        given, dout = dout, dout.reshape(-1, features)
        if dout.stride(1) != 1 and features > 1:
            dout = dout.contiguous()
        pack, codes = _setup()
        with _lib.on_device(dout):
            dweight = torch.empty(classes, features, dtype=dout.dtype, device=dout.device)
            head = (flat.numel(), padding_idx, classes, features, codes[dout.dtype], flat.dtype == torch.int64, scale, 0, flat.data_ptr(), 0, dout.data_ptr(), 0,
                    dweight.data_ptr(), 0, 0, dout.stride(0), features)
            work_bytes = _lib.lib().b200_embed_bwd_work_bytes(pack(*head, 0, 0))
            work = torch.empty(max(work_bytes, 1), dtype=torch.uint8, device=dout.device)
            _lib.call("b200_embed_bwd", pack(*head, work.data_ptr(), work_bytes), _lib.stream_of(dout))
            del work
        return None, *once((given,), (dweight,)), None, None


def token_embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: ids (...) int32 or int64, weight (classes, features) float32, float16 or
    bfloat16 -> (..., features).  The gradient of row ``padding_idx`` is zero.  An id outside
    [0, classes) reads nothing: its row is NaN, and it adds to no gradient.  Forward-mode derivatives are an error."""
    shape = weight.shape
    if len(shape) != 2 or 0 in shape:
        raise RuntimeError("token_embedding: weight (classes, features) expected")
    if weight.dtype not in _DT or not weight.is_cuda:
        raise RuntimeError("token_embedding: weight must be a float32 / float16 / bfloat16 CUDA tensor")
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise RuntimeError("token_embedding: ids must be int32 or int64")
    if ids.get_device() != weight.get_device():
        raise RuntimeError("token_embedding: ids and weight must be on one device")
    if padding_idx is None:
        padding_idx = -1
    elif -shape[0] <= padding_idx < shape[0]:
        padding_idx %= shape[0]
    else:
        raise RuntimeError("token_embedding: padding_idx must be a row of weight")
    if ids.numel() == 0:
        return weight[:0].sum() + weight.new_empty(ids.shape + (shape[1],))
    if recorded(weight):
        return TokenEmbeddingFn.apply(ids, weight, float(scale), padding_idx)
    return _lookup(ids, weight, *shape, float(scale), padding_idx)[0]
