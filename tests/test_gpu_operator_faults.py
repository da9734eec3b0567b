"""Calls of the loss without logits, the embedding and linear attention that were once answered wrongly, and what guards against each."""
from __future__ import annotations

import pytest
import torch

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
