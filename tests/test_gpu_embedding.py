"""Embedding lookup and its gradient against float64.

Forward: one product and one rounding (u = half a step of the type, and 2^-24 of the float32 product).  Backward: n rows
are added in float32, at most n 2^-24 of the sum of magnitudes, then scaled and rounded once.  Below 2^-14 float16 has steps of 2^-24 whatever the value, so half a step is at most 2^-25 there
(a single row of 1e-5 times sqrt(8) is such a gradient); TINY adds it."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DTYPES = list(HALF)


def ids_of(kind, tokens, classes, g):
    if kind == "uniform":
        return torch.randint(0, classes, (tokens,), generator=g)
    if kind == "one":
        return torch.full((tokens,), classes - 1)
    u = torch.rand(tokens, generator=g, dtype=torch.float64)
    return (torch.exp(u * torch.log(torch.tensor(classes + 1.0, dtype=torch.float64))) - 1).long().clamp(0, classes - 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "zipf", "one"])
@pytest.mark.parametrize("tokens,classes,features", [(1, 1, 1), (1, 50280, 64), (31, 5, 7), (32, 40, 8), (33, 512, 250), (2048, 511, 16), (2049, 513, 33),
                                                     (5000, 50280, 64), (20011, 300, 129), (4096, 262144, 8)])
def test_lookup_and_gradient(tokens, classes, features, kind, dtype):
    from lrnnx_b200.ops import token_embedding
    g = torch.Generator().manual_seed(tokens + classes * 3 + features)
    ids = ids_of(kind, tokens, classes, g).cuda()
    w = torch.randn(classes, features, generator=g).to(dtype).cuda().requires_grad_()
    dout = torch.randn(tokens, features, generator=g).to(dtype).cuda()
    u = HALF[dtype]
    out = token_embedding(ids, w)
    assert torch.equal(out, w[ids])
    for scale, pad in ((1.0, None), (features ** 0.5, 0)):
        out = token_embedding(ids, w, scale=scale, padding_idx=pad)
        want = w.detach().double()[ids] * scale
        assert bool(((out.double() - want).abs() <= (u + 2.0 ** -23) * want.abs() + TINY[dtype]).all())
        got, = torch.autograd.grad(out, w, dout)
        d = dout.double() * scale
        if pad is not None:
            d[ids == pad] = 0
        total = torch.zeros(classes, features, dtype=torch.float64, device="cuda").index_add_(0, ids, d)
        mag = torch.zeros_like(total).index_add_(0, ids, d.abs())
        n = torch.bincount(ids, minlength=classes).unsqueeze(1)
        bound = (n.clamp(max=300) + 4) * 2.0 ** -24 * mag + u * total.abs() + TINY[dtype]        # chains: 32 of a piece, then an eighth of the pieces, then 8
        assert got.dtype == dtype
        assert bool(((got.double() - total).abs() <= bound).all())
        assert torch.count_nonzero(got[n.squeeze(1) == 0]) == 0
        again, = torch.autograd.grad(token_embedding(ids, w, scale=scale, padding_idx=pad), w, dout)
        assert torch.equal(got, again)
