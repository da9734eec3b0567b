"""The loss without logits against the definition in float64 on the same operands.

Bounds, element by element.  u is half a step of the operands' type.  z: the tensor core adds 16 products at a time into
its float32 accumulator and truncates, at most 2^-23 of the running sum, so |dz| <= Z = (D / 16 + 8) 2^-23 |H| |W|^T (8: the
six products of a float32 split and what it leaves out).  A loss is off by at most 2 max Z and the error of exp, log and
the sum, 2^-21 (1 + |lse|).  dz is rounded to u of itself (float16 also to 2^-25 of the largest row weight), and multiplied
and summed in chains of at most 64 truncating steps a chain for float32 and rows / 16 otherwise; the result is rounded once.
"""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# half a step; a float32 split is exact to 2^-24 a factor and leaves out three products of at most 2^-24
HALF = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(rows, classes, features, dtype, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed * 1009 + rows + classes * 7 + features * 31)
    h = torch.randn(rows, features, generator=g).to(dtype)
    w = (torch.randn(classes, features, generator=g) * (spread / math.sqrt(features))).to(dtype)
    labels = torch.randint(0, classes, (rows,), generator=g)
    labels[torch.rand(rows, generator=g) < 0.2] = -100
    return h.cuda(), w.cuda(), labels.cuda()


def reference(h, w, labels, scale):
    """Losses, gradients and the sums of magnitudes their bounds go by; ``scale`` (rows): d result / d row loss."""
    h, w = h.double(), w.double()
    z = h @ w.t()
    lse = torch.logsumexp(z, 1)
    at = torch.arange(len(labels), device=h.device)
    ok = (labels >= 0) & (labels < w.shape[0])
    loss = torch.where(ok, lse - z[at, labels.clamp(0, w.shape[0] - 1)], 0.0)
    dz = torch.softmax(z, 1)
    Z = (h.abs() @ w.abs().t()).amax(1, keepdim=True) * (h.shape[1] / 16 + 8) * 2.0 ** -23
    p_err = dz * (2 * Z + 2.0 ** -21)
    dz[at[ok], labels[ok]] -= 1
    s = torch.where(ok, scale.double(), 0.0)
    return dict(loss=loss, lse=lse, Z=Z.squeeze(1), dz=dz * s[:, None], p_err=p_err * s.abs()[:, None], dh=(dz * s[:, None]) @ w, dw=(dz * s[:, None]).t() @ h,
                unit=float(s.abs().max()))


def check(got, ref, h, w, dtype):
    u = HALF[dtype]
    sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
    e = ref["p_err"] + u * ref["dz"].abs() + sub * ref["unit"]
    rows, classes = ref["dz"].shape
    for name, value, err, mag, n in (("dh", got[0], e @ w.double().abs(), ref["dz"].abs() @ w.double().abs(), classes),
                                     ("dw", got[1], e.t() @ h.double().abs(), ref["dz"].abs().t() @ h.double().abs(), rows)):
        if value is None:
            continue
        chain = min(n, 1024) if dtype == torch.float32 else n
        bound = err + (chain / 16 + 8) * 2.0 ** -23 * mag + u * ref[name].abs() + sub
        off = (value.double() - ref[name]).abs()
        assert value.dtype == dtype
        assert bool((off <= bound).all()), (name, float((off / bound.clamp(min=1e-300)).max()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,classes,features", [(1, 2, 1), (1, 1000, 64), (3, 255, 7), (128, 256, 64), (129, 257, 65), (200, 1000, 96), (64, 5000, 768),
                                                   (1500, 300, 72), (257, 50280, 40), (2100, 513, 264)])
def test_values_and_gradients(rows, classes, features, dtype):
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, labels = make(rows, classes, features, dtype)
    for reduction in ("mean", "none", "sum"):
        counted = max(1, int((labels != -100).sum()))
        if reduction == "none":
            up = torch.rand(rows, generator=torch.Generator().manual_seed(1)).cuda() * 2 - 0.5
            scale = up
        else:
            up = torch.tensor(1.75 * (rows if dtype == torch.float16 else 1), device="cuda")
            scale = (up.double() / (counted if reduction == "mean" else 1)).expand(rows)
        ref = reference(h, w, labels, scale)
        hh, ww = h.detach().requires_grad_(), w.detach().requires_grad_()
        loss = linear_cross_entropy(hh, ww, labels, reduction=reduction)
        assert loss.dtype == torch.float32
        row_bound = 2 * ref["Z"] + 2.0 ** -21 * (1 + ref["lse"].abs())
        if reduction == "none":
            assert bool(((loss.double() - ref["loss"]).abs() <= row_bound).all())
            assert torch.count_nonzero(loss[labels == -100]) == 0
        else:
            total = float(ref["loss"].sum()) / (counted if reduction == "mean" else 1)
            bound = float(row_bound.sum()) / (counted if reduction == "mean" else 1)
            assert abs(float(loss) - total) <= bound + 2.0 ** -24 * abs(total)
        got = torch.autograd.grad(loss, (hh, ww), up)
        check(got, ref, h, w, dtype)
        assert torch.count_nonzero(got[0][labels == -100]) == 0
