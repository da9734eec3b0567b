"""Calls of the loss without logits, the embedding and linear attention that were once answered wrongly, and what guards against each."""
from __future__ import annotations

import pytest
import torch

from test_gpu_linear_attention import HALF as ATTN_HALF, TINY, make as attn_operands, recurrence, with_gradients, within
from test_gpu_linear_cross_entropy import check, make as loss_operands, reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def fill_free_memory():
    """The allocator's free memory is one block of NaN, which the next workspaces are cut from."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.full((1 << 28,), float("nan"), device="cuda")
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ loss


# one piece of the vocabulary, a multiple of 256 classes rounded up has more stages of 64 than the classes themselves
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes,features", [(200, 5700, 96), (200, 8300, 96), (300, 10800, 200), (64, 17700, 64), (70, 27700, 40), (256, 51500, 8)])
def test_shared_contractions_add_up_what_was_written(rows, classes, features, dtype):
    """The blocks that share the contraction of dz W all write their sums, however the classes end: bounds as for any gradient."""
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, labels = loss_operands(rows, classes, features, dtype)
    hh, ww = h.detach().requires_grad_(), w.detach().requires_grad_()
    up = torch.tensor(float(rows), device="cuda")
    loss = linear_cross_entropy(hh, ww, labels)
    fill_free_memory()
    got = torch.autograd.grad(loss, (hh, ww), up)
    counted = int((labels != -100).sum())
    ref = reference(h, w, labels, torch.full((rows,), rows / counted, device="cuda", dtype=torch.float64))
    check(got, ref, h, w, dtype)


# ------------------------------------------------------------------------------------------------ linear attention


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("t", [0, 36, 37, 127, 150, 199])
def test_a_decay_reaches_no_earlier_step(t, value, dtype):
    """A decay that is infinite or NaN at a step is in no result before it, in no query's gradient before it and in no key's or
    value's gradient from it on; other heads and batch entries know nothing of it."""
    from lrnnx_b200.ops import linear_attention_fn
    (q, k, v, g, s0), dout, dlast = attn_operands(2, 200, 4, 2, 48, 64, dtype, "token", seed=14)
    zero = torch.zeros_like(s0)
    want = with_gradients((q, k, v, g, zero), 1.0, dout, torch.zeros_like(dlast))
    mag = with_gradients([x.abs() for x in (q, k, v)] + [g, zero], 1.0, dout.abs(), torch.zeros_like(dlast))
    bad = g.clone()
    bad[0, t, 1] = value
    leaves = [x.detach().requires_grad_() for x in (q, k, v, bad)]
    o = linear_attention_fn(*leaves)
    got = [o.detach(), *torch.autograd.grad(o, leaves, dout)]
    F, u, tiny = (200 / 16 + 200) * 2.0 ** -23, ATTN_HALF[dtype], TINY[dtype]
    for name, x, i, head, reached in (("o", got[0], 0, 1, slice(t, None)), ("dq", got[1], 2, 0, slice(t, None)), ("dk", got[2], 3, 0, slice(0, t)),
                                      ("dv", got[3], 4, 1, slice(0, t))):
        clean = torch.ones_like(x, dtype=torch.bool)
        clean[0, reached, head] = False                  # the first group is the first two heads
        within(name, x[clean], want[i][clean], ((F + 2 * u) * mag[i] + u * want[i].abs() + tiny)[clean])
