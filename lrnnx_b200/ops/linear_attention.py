"""Linear attention with a decay for each head (``b200_linattn_fwd / bwd / step``).

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,      out_t = scale S_t^T q_t

the matrix-state sibling of the selective scan (``selective_scan_fn``): a state of dk x dv for each head instead
of dstate for each channel, with the decay of a step given directly as its logarithm.  ``linear_attention_fn`` runs
whole sequences in chunks of matrix products, forward and backward; ``linear_attention_step`` advances a state by one
token in place, as ``selective_state_update`` does.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from .mamba_block import _DT, _stream

MAX_SIZE = 128            # of dk and dv


def _inner(t):
    """t with its last dimension contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _fill(a, q, k, v, g, scale, s0):
    a.batch, a.seqlen, a.groups, a.dk = q.shape
    a.heads, a.dv = v.shape[2:]
    a.dtype, a.g_dtype = _lib.enum(_DT[q.dtype]), _lib.enum(_DT[g.dtype])
    a.scale = scale
    a.q, a.k, a.v, a.g = q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr()
    a.q_bs, a.q_ls, a.q_hs, _ = q.stride()
    a.k_bs, a.k_ls, a.k_hs, _ = k.stride()
    a.v_bs, a.v_ls, a.v_hs, _ = v.stride()
    if g.dim() == 1:
        a.g_heads, a.g_hs = 1, g.stride(0)
    else:
        a.g_bs, a.g_ls, a.g_hs = g.stride()
    if s0 is not None:
        a.s0 = s0.data_ptr()
        a.s0_bs, a.s0_hs, a.s0_ks, _ = s0.stride()


def _work(a, name, like):
    a.work_bytes = getattr(_lib.lib(), name)(ctypes.byref(a))
    if not a.work_bytes:
        return None
    work = torch.empty(a.work_bytes, dtype=torch.uint8, device=like.device)
    a.work = work.data_ptr()
    return work


@functools.lru_cache(maxsize=None)
def _step_setup():
    return _lib.packer("b200_linattn_step_args"), {t: _lib.enum(n) for t, n in _DT.items()}


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, scale, initial_state, return_last_state):
        q, k, v = _inner(q), _inner(k), _inner(v)
        s0 = None if initial_state is None else _inner(initial_state)
        a = _lib.struct("b200_linattn_args")()
        _fill(a, q, k, v, g, scale, s0)
        last = None
        with _lib.on_device(q):
            out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
            a.out = out.data_ptr()
            a.out_bs, a.out_ls, a.out_hs, _ = out.stride()
            if return_last_state:
                last = torch.empty(a.batch, a.heads, a.dk, a.dv, dtype=torch.float32, device=v.device)
                a.last = last.data_ptr()
            work = _work(a, "b200_linattn_fwd_work_bytes", q)
            _lib.call("b200_linattn_fwd", a, _stream(q))
            del work
        ctx.save_for_backward(q, k, v, g, s0)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if return_last_state else out

    @staticmethod
    def backward(ctx, dout, dlast=None):
        q, k, v, g, s0 = ctx.saved_tensors
        if dout is None and dlast is None:
            return None, None, None, None, None, None, None
        a = _lib.struct("b200_linattn_args")()
        _fill(a, q, k, v, g, ctx.scale, s0)
        with _lib.on_device(q):
            dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if dout is None else _inner(dout)
            a.dout = dout.data_ptr()
            a.dout_bs, a.dout_ls, a.dout_hs, _ = dout.stride()
            if dlast is not None:
                dlast = dlast.contiguous()
                a.dlast = dlast.data_ptr()
            new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
            dq, dk, dv = new(q), new(k), new(v)
            a.dq, a.dk_out, a.dv_out = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
            dg = new(g) if ctx.needs_input_grad[3] else None
            ds0 = new(s0) if ctx.needs_input_grad[5] else None
            if dg is not None:
                a.dg = dg.data_ptr()
            if ds0 is not None:
                a.ds0 = ds0.data_ptr()
            work = _work(a, "b200_linattn_bwd_work_bytes", q)
            _lib.call("b200_linattn_bwd", a, _stream(q))
            del work
        return dq, dk, dv, dg, None, ds0, None


def _check(name, dims, q, k, v, g, state):
    batch, heads, dv = v.shape[0], v.shape[-2], v.shape[-1]
    if q.shape != k.shape or q.dim() != dims or v.dim() != dims or q.shape[:dims - 2] != v.shape[:dims - 2]:
        raise RuntimeError(f"{name}: q and k of one shape, v with the same batch{' and length' if dims == 4 else ''} expected")
    if q.shape[-2] == 0 or heads % q.shape[-2] != 0:
        raise RuntimeError(f"{name}: the heads of v must be a multiple of the groups of q and k")
    if not (1 <= q.shape[-1] <= MAX_SIZE and 1 <= dv <= MAX_SIZE):
        raise RuntimeError(f"{name}: head sizes must be 1 to {MAX_SIZE}")
    if tuple(g.shape) not in ((heads,), tuple(v.shape[:-1])):
        raise RuntimeError(f"{name}: g must be ({'batch, length, ' if dims == 4 else 'batch, '}heads) or (heads,)")
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype or g.dtype not in (torch.float32, q.dtype):
        raise RuntimeError(f"{name}: q, k and v must be float32 / float16 / bfloat16 of one dtype, g float32 or of that dtype")
    for t in (q, k, v, g, state):
        if t is not None and (not t.is_cuda or t.device != q.device):
            raise RuntimeError(f"{name}: all operands must be CUDA tensors on one device")


def linear_attention_fn(q, k, v, g, scale=1.0, initial_state=None, return_last_state=False):
    """q, k (batch, length, groups, dk), v (batch, length, heads, dv) of one dtype (float32, float16, bfloat16), any strides; heads a
    multiple of groups, dk and dv up to 128.  g: log decays, (batch, length, heads) or (heads,), float32 or the dtype of
    q; -inf starts from an empty state at that step (a new document).  ``initial_state`` float32 (batch, heads, dk, dv)
    is the state before the first step.  Returns out (batch, length, heads, dv), and with ``return_last_state`` the float32
    state after the last step.  Gradients for q, k, v, g and initial_state."""
    _check("linear_attention_fn", 4, q, k, v, g, initial_state)
    batch, length, heads, dv = v.shape
    if initial_state is not None and (tuple(initial_state.shape) != (batch, heads, q.shape[-1], dv) or initial_state.dtype != torch.float32):
        raise RuntimeError("linear_attention_fn: initial_state must be float32 (batch, heads, dk, dv)")
    if batch * heads > 65535:
        raise RuntimeError("linear_attention_fn: batch * heads must be at most 65535")
    if v.numel() == 0:                                    # no steps: nothing out, the state as it was
        out = v * 1 + (q.sum() + k.sum() + g[..., :0].sum()).to(v.dtype)
        if not return_last_state:
            return out
        return out, initial_state.clone() if initial_state is not None else torch.zeros(batch, heads, q.shape[-1], dv, device=v.device)
    return LinearAttentionFn.apply(q, k, v, g, float(scale), initial_state, return_last_state)


def linear_attention_step(state, q, k, v, g, scale=1.0, state_batch_indices=None):
    """One token: state (batch, heads, dk, dv), float32 or the dtype of q, dv contiguous, is updated in place; q, k (batch,
    groups, dk), v (batch, heads, dv), g (batch, heads) or (heads,).  With ``state_batch_indices`` (batch,) int32 the
    state is a pool and entry b advances slot ``state_batch_indices[b]``, no slot twice; an entry outside the pool has no
    state and gives zeros.  Returns out (batch, heads, dv).  No gradient; legal inside CUDA-graph capture."""
    _check("linear_attention_step", 3, q, k, v, g, state)
    batch, heads, dv = v.shape
    if state.dim() != 4 or tuple(state.shape[1:]) != (heads, q.shape[-1], dv) or state.stride(-1) != 1 and dv > 1:
        raise RuntimeError("linear_attention_step: state must be (batch, heads, dk, dv) with dv contiguous")
    if state.dtype not in (torch.float32, q.dtype):
        raise RuntimeError("linear_attention_step: the state must be float32 or of the dtype of q")
    if state_batch_indices is None:
        if state.shape[0] != batch:
            raise RuntimeError("linear_attention_step: state and q must have the same batch")
    elif (tuple(state_batch_indices.shape) != (batch,) or state_batch_indices.dtype != torch.int32 or not state_batch_indices.is_contiguous()
          or state_batch_indices.device != q.device):
        raise RuntimeError("linear_attention_step: state_batch_indices must be a contiguous int32 tensor (batch,) on the device of q")
    q, k, v = _inner(q), _inner(k), _inner(v)
    pack, codes = _step_setup()
    sq, sk, sv, sg, ss = q.stride(), k.stride(), v.stride(), g.stride(), state.stride()
    with _lib.on_device(q):
        out = torch.empty(batch, heads, dv, dtype=v.dtype, device=v.device)
        if batch == 0:
            return out
        _lib.call("b200_linattn_step",
                  pack(batch, heads, q.shape[1], q.shape[2], dv, codes[q.dtype], codes[g.dtype], codes[state.dtype], scale, state.shape[0], state.data_ptr(),
                       q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), 0 if state_batch_indices is None else state_batch_indices.data_ptr(),
                       out.data_ptr(), ss[0], ss[1], ss[2], sq[0], sq[1], sk[0], sk[1], sv[0], sv[1], sg[0] if g.dim() == 2 else 0, sg[-1], heads * dv, dv),
                  _lib.stream_of(q))
    return out
