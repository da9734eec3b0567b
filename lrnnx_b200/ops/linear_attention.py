"""Linear attention with a decay for each head (``b200_linattn_fwd / bwd / step``).

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,      out_t = scale S_t^T q_t

the matrix-state sibling of the selective scan (``selective_scan_fn``): a state of dk x dv for each head instead
of dstate for each channel, with the decay of a step given directly as its logarithm.  ``linear_attention_fn`` runs
whole sequences in chunks of matrix products, forward and backward; ``linear_attention_step`` advances a state by one
token in place, as ``selective_state_update`` does.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .mamba_block import _DT
from .once import once, recorded

MAX_SIZE = 128            # of dk and dv


def _inner(t):
    """t with its last dimension contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


@functools.lru_cache(maxsize=None)
def _setup():
    return _lib.packer("b200_linattn_args"), {t: _lib.enum(n) for t, n in _DT.items()}


def _call(name, q, k, v, g, scale, s0, out, last, back):
    """Runs b200_linattn_fwd or _bwd; ``back`` is the tail of the argument block that only the backward has."""
    pack, codes = _setup()
    batch, length, groups, dk = q.shape
    heads, dv = v.shape[2:]
    by_head = g.dim() == 1
    head = (batch, length, heads, groups, dk, dv, codes[q.dtype], codes[g.dtype], scale, by_head, q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(),
            0 if s0 is None else s0.data_ptr(), out, last, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
            *((0, 0, g.stride(0)) if by_head else g.stride()), *((0, 0, 0) if s0 is None else s0.stride()[:3]), length * heads * dv, heads * dv, dv, *back)
    lib = _lib.lib()
    work_bytes = getattr(lib, name + "_work_bytes")(pack(*head, 0, 0))
    work = torch.empty(work_bytes, dtype=torch.uint8, device=q.device) if work_bytes else None
    _lib.call(name, pack(*head, work.data_ptr() if work_bytes else 0, work_bytes), _lib.stream_of(q))


@functools.lru_cache(maxsize=None)
def _step_setup():
    return _lib.packer("b200_linattn_step_args"), {t: _lib.enum(n) for t, n in _DT.items()}


def _forward(q, k, v, g, scale, s0, return_last_state):
    with _lib.on_device(q):
        out = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        last = torch.empty((v.shape[0], v.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32, device=v.device) if return_last_state else None
        _call("b200_linattn_fwd", q, k, v, g, scale, s0, out.data_ptr(), last.data_ptr() if return_last_state else 0, (0,) * 10)
    return out, last


class LinearAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, scale, initial_state, return_last_state):
        q, k, v = _inner(q), _inner(k), _inner(v)
        s0 = None if initial_state is None else _inner(initial_state)
        out, last = _forward(q, k, v, g, scale, s0, return_last_state)
        ctx.save_for_backward(q, k, v, g, s0)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (out, last) if return_last_state else out

    @staticmethod
    def backward(ctx, dout, dlast=None):
        q, k, v, g, s0 = ctx.saved_tensors
        if dout is None and dlast is None:
            return None, None, None, None, None, None, None
        given = [t for t in (q, k, v, g, s0, dout, dlast) if t is not None]
        new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        with _lib.on_device(q):
            dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device) if dout is None else _inner(dout)
            dlast = None if dlast is None else dlast.contiguous()
            dq, dk, dv = new(q), new(k), new(v)
            dg = new(g) if ctx.needs_input_grad[3] else None
            ds0 = new(s0) if ctx.needs_input_grad[5] else None
            at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
            _call("b200_linattn_bwd", q, k, v, g, ctx.scale, s0, 0, 0,
                  (dout.data_ptr(), at(dlast), *dout.stride()[:3], dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), at(dg), at(ds0)))
        dq, dk, dv, dg, ds0 = once(given, (dq, dk, dv, dg, ds0))
        return dq, dk, dv, dg, None, ds0, None


def _check(name, dims, q, k, v, g, state):
    qs, vs, gs = q.shape, v.shape, g.shape
    if len(qs) != dims or qs != k.shape or len(vs) != dims or qs[:dims - 2] != vs[:dims - 2]:
        raise RuntimeError(f"{name}: q and k of one shape, v with the same batch{' and length' if dims == 4 else ''} expected")
    heads, dv = vs[-2:]
    if qs[-2] == 0 or heads % qs[-2] != 0:
        raise RuntimeError(f"{name}: the heads of v must be a multiple of the groups of q and k")
    if not (1 <= qs[-1] <= MAX_SIZE and 1 <= dv <= MAX_SIZE):
        raise RuntimeError(f"{name}: head sizes must be 1 to {MAX_SIZE}")
    if gs != vs[:-1] and (len(gs) != 1 or gs[0] != heads):
        raise RuntimeError(f"{name}: g must be ({'batch, length, ' if dims == 4 else 'batch, '}heads) or (heads,)")
    dtype = q.dtype
    if dtype not in _DT or k.dtype != dtype or v.dtype != dtype or g.dtype != dtype and g.dtype != torch.float32:
        raise RuntimeError(f"{name}: q, k and v must be float32 / float16 / bfloat16 of one dtype, g float32 or of that dtype")
    device = q.get_device()
    if device < 0 or k.get_device() != device or v.get_device() != device or g.get_device() != device or state is not None and state.get_device() != device:
        raise RuntimeError(f"{name}: all operands must be CUDA tensors on one device")


def linear_attention_fn(q, k, v, g, scale=1.0, initial_state=None, return_last_state=False):
    """q, k (batch, length, groups, dk), v (batch, length, heads, dv) of one dtype (float32, float16, bfloat16), any strides; heads a
    multiple of groups, dk and dv up to 128.  g: log decays, (batch, length, heads) or (heads,), float32 or the dtype of
    q; -inf starts from an empty state at that step (a new document; the state is multiplied by zero, so that one that is
    not finite is NaN from there).  ``initial_state`` float32 (batch, heads, dk, dv) is the state before the first step.
    Returns out (batch, length, heads, dv), and with ``return_last_state`` the float32 state after the last step.  An
    infinite or NaN value reaches its own step and later ones, no earlier result.  Gradients for q, k, v, g and
    initial_state; forward-mode derivatives are an error."""
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
    # copies that the kernels need are made here, where autograd sees them: what is saved is then what came in, which second derivatives go by
    q, k, v, s0 = _inner(q), _inner(k), _inner(v), None if initial_state is None else _inner(initial_state)
    if recorded(q, k, v, g, s0):
        return LinearAttentionFn.apply(q, k, v, g, float(scale), s0, return_last_state)
    out, last = _forward(q, k, v, g, float(scale), s0, return_last_state)
    return (out, last) if return_last_state else out


def linear_attention_step(state, q, k, v, g, scale=1.0, state_batch_indices=None):
    """One token: state (batch, heads, dk, dv), float32 or the dtype of q, dv contiguous, is updated in place; q, k (batch,
    groups, dk), v (batch, heads, dv), g (batch, heads) or (heads,).  With ``state_batch_indices`` (batch,) int32 the
    state is a pool and entry b advances slot ``state_batch_indices[b]``, no slot twice (blocks would race for it); an
    entry outside the pool has no state and gives zeros.  A decay of -inf multiplies the state by zero: a slot to be used
    anew that may hold anything is cleared first.  Returns out (batch, heads, dv).  No gradient; legal inside CUDA-graph
    capture."""
    _check("linear_attention_step", 3, q, k, v, g, state)
    batch, heads, dv = v.shape
    _, groups, dk = q.shape
    slots, ss = state.shape[0], state.stride()
    if state.shape[1:] != (heads, dk, dv) or ss[3] != 1 and dv > 1:
        raise RuntimeError("linear_attention_step: state must be (batch, heads, dk, dv) with dv contiguous")
    if 0 in ss and any(x == 0 and n > 1 for x, n in zip(ss, state.shape)):
        raise RuntimeError("linear_attention_step: elements of the state must not share memory, it is updated in place")
    if state.dtype != q.dtype and state.dtype != torch.float32:
        raise RuntimeError("linear_attention_step: the state must be float32 or of the dtype of q")
    if state_batch_indices is None:
        if slots != batch:
            raise RuntimeError("linear_attention_step: state and q must have the same batch")
    elif (state_batch_indices.shape != (batch,) or state_batch_indices.dtype != torch.int32 or not state_batch_indices.is_contiguous()
          or state_batch_indices.get_device() != q.get_device()):
        raise RuntimeError("linear_attention_step: state_batch_indices must be a contiguous int32 tensor (batch,) on the device of q")
    q, k, v = _inner(q), _inner(k), _inner(v)
    pack, codes = _step_setup()
    sq, sk, sv, sg = q.stride(), k.stride(), v.stride(), g.stride()
    with _lib.on_device(q):
        out = v.new_empty((batch, heads, dv))
        if batch == 0:
            return out
        _lib.call("b200_linattn_step",
                  pack(batch, heads, groups, dk, dv, codes[q.dtype], codes[g.dtype], codes[state.dtype], float(scale), slots, state.data_ptr(),
                       q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), 0 if state_batch_indices is None else state_batch_indices.data_ptr(),
                       out.data_ptr(), ss[0], ss[1], ss[2], sq[0], sq[1], sk[0], sk[1], sv[0], sv[1], sg[0] if len(sg) == 2 else 0, sg[-1], heads * dv, dv),
                  _lib.stream_of(q))
    return out
