"""The language model's embedding module where nn.Embedding's own path answers: on the CPU (here), and with its options (on a GPU)."""
from __future__ import annotations

import pytest
import torch
import torch.nn as nn

from lrnnx_b200.lm import MambaLMHeadModel, TokenEmbedding


def _pair(device="cpu", dtype=None, **kw):
    torch.manual_seed(3)
    ours, theirs = TokenEmbedding(12, 6, device=device, dtype=dtype, **kw), nn.Embedding(12, 6, device=device, dtype=dtype, **kw)
    with torch.no_grad():
        theirs.weight.copy_(ours.weight)
    return ours, theirs, torch.tensor([[1, 2, 2], [11, 0, 2]], device=device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("kw", [{}, {"padding_idx": 2}, {"max_norm": 1.0}, {"scale_grad_by_freq": True}, {"sparse": True}])
def test_as_nn_embedding_on_the_cpu(kw, dtype):
    ours, theirs, ids = _pair(dtype=dtype, **kw)
    a, b = ours(ids), theirs(ids)
    assert torch.equal(a, b)
    a.sum().backward()
    b.sum().backward()
    assert ours.weight.grad.is_sparse == theirs.weight.grad.is_sparse
    assert torch.equal(ours.weight.grad.to_dense(), theirs.weight.grad.to_dense())


def test_from_pretrained_and_the_models_own():
    w = torch.randn(7, 4)
    m = TokenEmbedding.from_pretrained(w, freeze=False)
    assert type(m) is TokenEmbedding and m.weight.requires_grad and torch.equal(m(torch.tensor([6, 0])), w[[6, 0]])
    model = MambaLMHeadModel(16, 1, 20)
    ids = torch.tensor([[3, 19]])
    assert torch.equal(model.backbone.embedding(ids), model.lm_head.weight[ids])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{"max_norm": 1.0}, {"scale_grad_by_freq": True}, {"sparse": True}, {"padding_idx": 2}, {}])
def test_options_on_a_gpu(kw):
    """Small whole numbers as gradients: sums are exact in any order."""
    ours, theirs, ids = _pair("cuda", **kw)
    a, b = ours(ids), theirs(ids)
    assert torch.equal(a, b)
    a.sum().backward()
    b.sum().backward()
    assert ours.weight.grad.is_sparse == theirs.weight.grad.is_sparse
    x, y = ours.weight.grad.to_dense(), theirs.weight.grad.to_dense()
    assert torch.equal(x, y) if "scale_grad_by_freq" not in kw else bool(((x - y).abs() <= 2.0 ** -22 * y.abs()).all())


@pytest.mark.gpu
def test_weights_in_64_bits_on_a_gpu():
    ours, theirs, ids = _pair("cuda", dtype=torch.float64)
    assert torch.equal(ours(ids), theirs(ids))
