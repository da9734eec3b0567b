"""Edges of the loss without logits, the embedding and linear attention: operands as views (inside NaN, at odd offsets, transposed,
broadcast), labels and ids that mean nothing, empty and one-step calls, single gradients, more than one piece of the
vocabulary, another stream, captured calls, the same bits twice, and a model that runs them together."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from test_gpu_linear_attention import HALF as ATTN_HALF, TINY, make as attn_operands, recurrence, with_gradients, within
from test_gpu_linear_cross_entropy import check, make as loss_operands, reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def moat(t, pad):
    """A view equal to t inside NaN, ``pad`` elements on both sides of its last dimension."""
    big = torch.full(tuple(t.shape[:-1]) + (t.shape[-1] + 2 * pad,), float("nan"), dtype=t.dtype, device=t.device)
    view = big[..., pad:pad + t.shape[-1]]
    view.copy_(t)
    return view


# ------------------------------------------------------------------------------------------------ loss


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad", [8, 3])             # rows that TMA reads in place, rows that are packed first
def test_loss_reads_views(dtype, pad):
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, labels = loss_operands(150, 700, 72, dtype)
    want = linear_cross_entropy(h, w, labels, reduction="none")
    hv, wv = moat(h, pad).requires_grad_(), moat(w, pad).requires_grad_()
    got = linear_cross_entropy(hv, wv, labels, reduction="none")
    assert torch.equal(got, want)
    up = torch.rand(150, device="cuda")
    a = torch.autograd.grad(got, (hv, wv), up)
    b = torch.autograd.grad(linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), labels, reduction="none"), (h, w), up)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # transposed operands, three dimensions, 32-bit labels
    got = linear_cross_entropy(h.detach().t().contiguous().t().view(150, 72), w.detach().t().contiguous().t(), labels.int(), reduction="none")
    assert torch.equal(got, want)
    got = linear_cross_entropy(h.detach().view(10, 15, 72), w, labels.view(10, 15), reduction="none")
    assert got.shape == (10, 15) and torch.equal(got.flatten(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_labels_that_mean_nothing(dtype):
    """Labels outside the classes have no loss and no gradient and count in the mean, as in cross_entropy; ignored rows hold no
    part even where they are the only ones."""
    from lrnnx_b200.ops import linear_cross_entropy
    from lrnnx_b200.ops.cross_entropy import cross_entropy
    h, w, labels = loss_operands(40, 300, 64, dtype)
    labels[3], labels[4], labels[5] = 300, -7, 1 << 40
    hh, ww = h.requires_grad_(), w.requires_grad_()
    loss = linear_cross_entropy(hh, ww, labels)
    logits = h.detach().float() @ w.detach().float().t()
    assert abs(float(loss.detach()) - float(cross_entropy(logits, labels))) <= 2.0 ** -17 * (1 + float(loss.detach()))
    dh, dw = torch.autograd.grad(loss, (hh, ww))
    assert torch.count_nonzero(dh[3:6]) == 0 and torch.count_nonzero(dh[labels == -100]) == 0
    none = linear_cross_entropy(hh, ww, torch.full((40,), -100, device="cuda"))
    assert float(none.detach()) == 0.0
    dh, dw = torch.autograd.grad(none, (hh, ww))
    assert torch.count_nonzero(dh) == 0 and torch.count_nonzero(dw) == 0
    assert float(linear_cross_entropy(h.detach(), w.detach(), labels.clamp(0, 299), ignore_index=0, reduction="sum")) > 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_each_gradient_alone_and_bits_twice(dtype):
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, labels = loss_operands(600, 2000, 320, dtype)
    both = torch.autograd.grad(linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), labels), (h, w))
    for _ in range(2):
        dh, = torch.autograd.grad(linear_cross_entropy(h, w.detach(), labels), h)
        dw, = torch.autograd.grad(linear_cross_entropy(h.detach(), w, labels), w)
        assert torch.equal(dh, both[0]) and torch.equal(dw, both[1])


@pytest.mark.parametrize("dtype,rows,classes,features", [(torch.bfloat16, 70001, 9001, 24), (torch.float32, 30011, 8200, 40)])
def test_vocabulary_in_pieces(dtype, rows, classes, features):
    """More rows x classes than one piece of the logits' gradient holds; the memory taken stays below the logits'."""
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, labels = loss_operands(rows, classes, features, dtype)
    hh, ww = h.requires_grad_(), w.requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss = linear_cross_entropy(hh, ww, labels)
    got = torch.autograd.grad(loss, (hh, ww), torch.tensor(float(rows), device="cuda"))
    peak = torch.cuda.max_memory_allocated() - before
    assert peak < (1 << 30) + (1 << 28) and peak < 4 * rows * classes
    counted = int((labels != -100).sum())
    ref = reference(h.detach(), w.detach(), labels, torch.full((rows,), rows / counted, device="cuda", dtype=torch.float64))
    check(got, ref, h.detach(), w.detach(), dtype)


def test_loss_gradient_against_differences():
    """Float32, a direction in weight and hidden: the loss is smooth, a step of 2^-7 leaves an error of its third derivative's
    order, 2^-14 of a slope of order one, and 2^-20 / 2^-7 of the loss's rounding."""
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, labels = loss_operands(64, 500, 48, torch.float32)
    dh, dw = torch.autograd.grad(linear_cross_entropy(h.requires_grad_(), w.requires_grad_(), labels), (h, w))
    g = torch.Generator(device="cuda").manual_seed(1)
    for t, d, f in ((h, dh, lambda x: linear_cross_entropy(x, w.detach(), labels)), (w, dw, lambda x: linear_cross_entropy(h.detach(), x, labels))):
        u = torch.randn(t.shape, generator=g, device="cuda")
        e = 2.0 ** -7
        num = (float(f(t.detach() + e * u)) - float(f(t.detach() - e * u))) / (2 * e)
        assert abs(num - float((d * u).sum())) <= 2e-3


# ------------------------------------------------------------------------------------------------ embedding


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_views_and_bad_ids(dtype):
    from lrnnx_b200.ops import token_embedding
    g = torch.Generator().manual_seed(3)
    w = torch.randn(50, 40, generator=g).to(dtype).cuda()
    ids = torch.randint(0, 50, (7, 9), generator=g).cuda()
    want = w[ids]
    for pad in (8, 4, 3, 1):
        assert torch.equal(token_embedding(ids, moat(w, pad)), want)
    assert torch.equal(token_embedding(ids.int(), w), want)
    assert torch.equal(token_embedding(ids.t(), w), want.transpose(0, 1))
    assert torch.equal(token_embedding(ids, w.t().contiguous().t()), want)
    assert token_embedding(ids[:0], w).shape == (0, 9, 40)
    # ids without a row: NaN, and no part in the gradient
    bad = ids.clone()
    bad[0, 0], bad[1, 1], bad[2, 2] = -1, 50, 1 << 40
    ww = w.clone().requires_grad_()
    out = token_embedding(bad, ww)
    assert bool(torch.isnan(out[0, 0]).all() and torch.isnan(out[1, 1]).all() and torch.isnan(out[2, 2]).all())
    ok = torch.ones(7, 9, dtype=torch.bool)
    ok[0, 0] = ok[1, 1] = ok[2, 2] = False
    assert torch.equal(out[ok.cuda()], want[ok.cuda()])
    dout = torch.randn(7, 9, 40, generator=g).to(dtype).cuda()
    got, = torch.autograd.grad(out, ww, dout)
    alone = w.clone().requires_grad_()
    want_g, = torch.autograd.grad(token_embedding(ids[ok.cuda()], alone), alone, dout[ok.cuda()])
    assert torch.equal(got, want_g)
    # gradients that come in transposed, broadcast, and inside NaN
    for d in (dout.transpose(0, 1).contiguous().transpose(0, 1), moat(dout, 8), moat(dout, 1)):
        assert torch.equal(torch.autograd.grad(token_embedding(ids, ww), ww, d)[0], torch.autograd.grad(token_embedding(ids, ww), ww, dout)[0])
    one, = torch.autograd.grad(token_embedding(ids, ww).sum(), ww)
    assert torch.equal(one, torch.bincount(ids.flatten(), minlength=50).to(dtype).unsqueeze(1).expand(50, 40))


# ------------------------------------------------------------------------------------------------ linear attention


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["projection", "heads_first", "odd", "broadcast"])
def test_attention_reads_any_strides(layout, dtype):
    """Slices of one projection, (batch, heads, length) tensors, rows at odd offsets inside NaN, and operands broadcast over the batch."""
    from lrnnx_b200.ops import linear_attention_fn
    (q, k, v, g, s0), dout, dlast = attn_operands(2, 150, 4, 4, 64, 64, dtype, "token", seed=2)
    if layout == "broadcast":
        q, v, g, s0 = q[:1].expand(2, -1, -1, -1), v[:, :, :1].expand(-1, -1, 4, -1), g[:1].expand(2, -1, -1), s0[:, :1].expand(-1, 4, -1, -1)
    dense = [t.contiguous() for t in (q, k, v, g, s0)]
    if layout == "projection":
        x = torch.stack([q, k, v], 3).flatten(2)
        q, k, v = x.view(2, 150, 4, 3, 64).unbind(3)
    elif layout == "heads_first":
        q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
        g, s0, dout = g.transpose(1, 2).contiguous().transpose(1, 2), s0.transpose(2, 3).contiguous().transpose(2, 3), dout.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "odd":
        q, k, v, g, s0, dout = (moat(t, 3) for t in (q, k, v, g, s0, dout))
    res = []
    for ops in ((q, k, v, g, s0), dense):
        leaves = [t.detach().requires_grad_() for t in ops]
        o, last = linear_attention_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
        res.append([o, last] + list(torch.autograd.grad([o, last], leaves, [dout, dlast])))
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_partial_calls(dtype):
    """No steps, no batch, one output's gradient at a time, a decay of the operands' type, a decay without a gradient, no growth and growth."""
    from lrnnx_b200.ops import linear_attention_fn
    (q, k, v, g, s0), dout, dlast = attn_operands(2, 70, 2, 1, 16, 24, dtype, "token", seed=4)
    o, last = linear_attention_fn(q[:, :0], k[:, :0], v[:, :0], g[:, :0], initial_state=s0, return_last_state=True)
    assert o.shape == (2, 0, 2, 24) and torch.equal(last, s0)
    assert linear_attention_fn(q[:0], k[:0], v[:0], g[:0]).shape == (0, 70, 2, 24)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, s0)]
    o, last = linear_attention_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
    whole = torch.autograd.grad([o, last], leaves, [dout, dlast], retain_graph=True)
    a = torch.autograd.grad(o, leaves, dout, retain_graph=True)
    b = torch.autograd.grad(last, leaves, dlast, retain_graph=True)
    none = torch.zeros_like(dout)
    assert all(torch.equal(x, y) for x, y in zip(b, torch.autograd.grad([o, last], leaves, [none, dlast])))
    for w, x, y in zip(whole, a, b):
        scale = float(w.double().abs().max())
        assert float((w.double() - x.double() - y.double()).abs().max()) <= (4 * ATTN_HALF[dtype] + 2.0 ** -16) * scale * 4
    no_g = linear_attention_fn(leaves[0], k, v, g)
    dq, = torch.autograd.grad(no_g, leaves[0], dout)
    only = linear_attention_fn(*[t.detach() for t in (q, k, v, g)])
    assert torch.equal(only, no_g)
    # decays of the operands' type, and one that grows
    g16 = g.to(dtype).requires_grad_()
    o, = [linear_attention_fn(q, k, v, g16)]
    dg, = torch.autograd.grad(o, g16, dout)
    assert dg.dtype == dtype
    assert torch.equal(o, linear_attention_fn(q, k, v, g16.detach().float()))
    up = torch.full((2,), 0.01, device="cuda")
    want, _ = recurrence(q.double(), k.double(), v.double(), up.double(), 1.0, torch.zeros(2, 2, 16, 24, dtype=torch.float64, device="cuda"))
    mag, _ = recurrence(q.double().abs(), k.double().abs(), v.double().abs(), up.double(), 1.0, torch.zeros(2, 2, 16, 24, dtype=torch.float64, device="cuda"))
    within("growth", linear_attention_fn(q, k, v, up), want, (204 * 2.0 ** -23 + 3 * ATTN_HALF[dtype]) * mag + TINY[dtype])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1100, 2400])
def test_attention_over_several_borders(n, dtype):
    """Segments, and more than two of the borders (every 512 steps) that the decays' gradient is anchored at."""
    from lrnnx_b200.ops import linear_attention_fn
    (q, k, v, g, s0), dout, dlast = attn_operands(1, n, 2, 2, 32, 40, dtype, "head", seed=6)
    g = (g / 50).contiguous()
    want = with_gradients((q, k, v, g, s0), 0.5, dout, dlast)
    mag = with_gradients([t.abs() for t in (q, k, v)] + [g, s0.abs()], 0.5, dout.abs(), dlast.abs())
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, s0)]
    o, last = linear_attention_fn(*leaves[:4], scale=0.5, initial_state=leaves[4], return_last_state=True)
    got = [o, last] + list(torch.autograd.grad([o, last], leaves, [dout, dlast]))
    F_, u = (n / 16 + 200) * 2.0 ** -23, ATTN_HALF[dtype]
    for i in (0, 2, 3, 4):
        within(str(i), got[i], want[i], (F_ + 2 * u) * mag[i] + u * want[i].abs())
    for i in (1, 6):
        within(str(i), got[i], want[i], F_ * mag[i])
    assert float((got[5].double() - want[5]).norm() / want[5].norm()) <= 1e-5


def test_attention_gradient_against_differences():
    """Float32: the result is linear in q, k, v and the state, so a difference is its gradient up to rounding; a decay's slope is
    taken over 2^-7, with an error of the order of its square."""
    from lrnnx_b200.ops import linear_attention_fn
    (q, k, v, g, s0), dout, _ = attn_operands(2, 90, 2, 1, 16, 16, torch.float32, "token", seed=8)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, s0)]
    grads = torch.autograd.grad((linear_attention_fn(*leaves[:4], initial_state=leaves[4]) * dout).sum(), leaves)
    gen = torch.Generator(device="cuda").manual_seed(2)
    for i in range(5):
        u = torch.randn(leaves[i].shape, generator=gen, device="cuda")
        e = 2.0 ** -7 if i == 3 else 0.5
        vals = []
        for sign in (1, -1):
            x = [t.detach() for t in leaves]
            x[i] = x[i] + sign * e * u
            vals.append(float((linear_attention_fn(*x[:4], initial_state=x[4]).double() * dout.double()).sum()))
        num, want = (vals[0] - vals[1]) / (2 * e), float((grads[i] * u).sum())
        assert abs(num - want) <= (1e-2 if i == 3 else 1e-4) * max(1.0, float((grads[i] * u).abs().sum()))


def test_step_in_a_pool_past_32_bits():
    """A slot whose elements begin beyond 2^31."""
    from lrnnx_b200.ops import linear_attention_step
    heads, dk, dv = 8, 128, 128
    slots = (1 << 31) // (heads * dk * dv) + 3
    pool = torch.empty(slots, heads, dk, dv, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([slots - 1, 0], dtype=torch.int32, device="cuda")
    pool[slots - 1], pool[0] = 1.0, 2.0
    (q, k, v, g, _), _, _ = attn_operands(2, 1, heads, heads, dk, dv, torch.bfloat16, "token")
    out = linear_attention_step(pool, q[:, 0], k[:, 0], v[:, 0], g[:, 0], state_batch_indices=at)
    small = torch.stack([torch.full((heads, dk, dv), c, dtype=torch.bfloat16, device="cuda") for c in (1.0, 2.0)])
    want = linear_attention_step(small, q[:, 0], k[:, 0], v[:, 0], g[:, 0])
    assert torch.equal(out, want) and torch.equal(pool[at.long()], small)


# ------------------------------------------------------------------------------------------------ streams, graphs, together


def _train(h, w, labels, ids, q, k, v, g, dout):
    from lrnnx_b200.ops import linear_attention_fn, linear_cross_entropy, token_embedding
    loss = linear_cross_entropy(h, w, labels)
    o = linear_attention_fn(q, k, v, g)
    e = token_embedding(ids, w)
    return [loss.detach(), o.detach()] + list(torch.autograd.grad([loss, o, e], [h, w, q, k, v, g], [None, dout, torch.ones_like(e)]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_on_another_stream(dtype):
    """Forward and backward recorded once and replayed on new values, two graphs alive together, and the same calls on a side stream."""
    (q, k, v, g, _), dout, _ = attn_operands(2, 300, 4, 2, 64, 64, dtype, "token", seed=9)
    h, w, labels = loss_operands(200, 1000, 64, dtype)
    ids = torch.randint(0, 1000, (2, 50), device="cuda")
    leaves = [t.requires_grad_() for t in (h, w, q, k, v, g)]
    args = lambda: (leaves[0], leaves[1], labels, ids, *leaves[2:], dout)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            on_side = _train(*args())
    torch.cuda.current_stream().wait_stream(side)
    want = _train(*args())
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    del on_side, want
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = _train(*args())
        graphs.append((graph, out))
    with torch.no_grad():
        for t in leaves[:5]:
            t.mul_(0.5)
        labels.copy_(labels.roll(1))
        ids.copy_((ids + 1) % 1000)
    for graph, _ in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    held = [[t.clone() for t in out] for _, out in graphs]
    now = _train(*args())
    for out in held:
        assert all(torch.equal(a, b) for a, b in zip(out, now))


def test_step_captured():
    from lrnnx_b200.ops import linear_attention_step
    (q, k, v, g, _), _, _ = attn_operands(3, 8, 4, 4, 64, 32, torch.bfloat16, "token", seed=12)
    state, again = torch.zeros(3, 4, 64, 32, device="cuda"), torch.zeros(3, 4, 64, 32, device="cuda")
    bufs = [t[:, 0].clone() for t in (q, k, v, g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        linear_attention_step(state, *bufs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = linear_attention_step(state, *bufs)
    state.zero_()
    for t in range(8):
        for b, x in zip(bufs, (q, k, v, g)):
            b.copy_(x[:, t])
        graph.replay()
        want = linear_attention_step(again, *[x[:, t] for x in (q, k, v, g)])
        assert torch.equal(out, want) and torch.equal(state, again)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_model_loss_is_the_loss_of_its_logits(dtype):
    """MambaLMHeadModel.loss against cross_entropy of the logits, with all gradients; tied weights take both ends' parts."""
    from lrnnx_b200.lm import MambaLMHeadModel
    from lrnnx_b200.ops.cross_entropy import cross_entropy
    torch.manual_seed(0)
    m = MambaLMHeadModel(64, 2, 500, device="cuda", dtype=dtype)
    ids = torch.randint(0, 500, (2, 40), device="cuda")
    labels = F.pad(ids[:, 1:], (0, 1), value=-100)
    params = [p for p in m.parameters()]
    a = m.loss(ids, labels)
    b = cross_entropy(m(ids).view(-1, 500), labels.view(-1))
    # logits of the second are rounded to the type, half a step of values up to 2 at most; means of losses around log 500
    assert abs(float(a.detach()) - float(b.detach())) <= (2.0 ** -18 if dtype == torch.float32 else 2.0 ** -7)
    ga, gb = torch.autograd.grad(a, params), torch.autograd.grad(b, params)
    for (n, p), x, y in zip(m.named_parameters(), ga, gb):
        # float32: sums of a few thousand products in another order; bfloat16: roundings of logits, hidden states and gradients
        assert x.dtype == p.dtype
        assert float((x.double() - y.double()).norm()) <= (2e-5 if dtype == torch.float32 else 3e-2) * float(y.double().norm()) + 1e-12, n


def test_embedding_mixer_and_loss_together():
    """A one-layer model with tied weights, lookup -> linear attention -> loss, float32: loss and gradients against the same model
    in float64 by its definition.  Relative 2-norms: products of three stages with at most 200 float32 roundings a sum, 2^-23 each."""
    from lrnnx_b200.ops import linear_attention_fn, linear_cross_entropy, token_embedding
    gen = torch.Generator().manual_seed(11)
    V, D, H, L, B = 311, 48, 3, 100, 2
    w = (torch.randn(V, D, generator=gen) * 0.3).cuda()
    p = [(torch.randn(D, D, generator=gen) / math.sqrt(D)).cuda() for _ in range(3)] + [(torch.randn(H, D, generator=gen) / math.sqrt(D)).cuda()]
    ids = torch.randint(0, V, (B, L), generator=gen).cuda()
    labels = F.pad(ids[:, 1:], (0, 1), value=-100)

    def model(w, p, embed, mix, loss):
        x = embed(ids, w)
        q, k, v = ((x @ m).view(B, L, H, D // H) for m in p[:3])
        g = -F.softplus(x @ p[3].t())
        return loss(x + mix(q, k, v, g).reshape(B, L, D), w)

    ours = [t.clone().requires_grad_() for t in [w] + p]
    a = model(ours[0], ours[1:], lambda i, w: token_embedding(i, w, scale=2.0), lambda *t: linear_attention_fn(*t, scale=0.25), lambda x, w: linear_cross_entropy(x, w, labels))
    exact = [t.double().requires_grad_() for t in [w] + p]
    zero = torch.zeros(B, H, D // H, D // H, dtype=torch.float64, device="cuda")
    b = model(exact[0], exact[1:], lambda i, w: 2.0 * w[i], lambda q, k, v, g: recurrence(q, k, v, g, 0.25, zero)[0],
              lambda x, w: F.cross_entropy((x @ w.t()).view(-1, V), labels.view(-1)))
    assert abs(float(a.detach()) - float(b.detach())) <= 200 * 2.0 ** -23 * (1 + float(b.detach()))
    for x, y in zip(torch.autograd.grad(a, ours), torch.autograd.grad(b, exact)):
        assert float((x.double() - y).norm()) <= 3 * 200 * 2.0 ** -23 * float(y.norm())


# ------------------------------------------------------------------------------------------------ what is masked stays out


@pytest.mark.parametrize("dtype", DTYPES)
def test_ignored_rows_may_hold_anything(dtype):
    """NaN and infinities in the hidden states of rows without a label (the padding of a batch) are in no result."""
    from lrnnx_b200.ops import linear_cross_entropy
    for pad in (None, 3):
        h, w, labels = loss_operands(140, 500, 72, dtype)
        labels[5], labels[6], labels[139] = -100, 500, -100
        bad = h.clone()
        bad[labels == -100], bad[6] = float("nan"), float("inf")
        zero = h.clone()
        zero[labels == -100], zero[6] = 0, 0
        res = []
        for x in (bad, zero):
            x = (x if pad is None else moat(x, pad)).requires_grad_()
            ww = w.clone().requires_grad_()
            loss = linear_cross_entropy(x, ww, labels)
            res.append([loss.detach(), *torch.autograd.grad(loss, (x, ww))])
        assert bool(torch.isfinite(res[0][2]).all()) and torch.count_nonzero(res[0][1][labels == -100]) == 0
        assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_is_causal_whatever_comes_later(dtype, value):
    """Values, keys and queries that are infinite or NaN at a step reach no earlier step, and a value only its own column."""
    from lrnnx_b200.ops import linear_attention_fn
    (q, k, v, g, _), _, _ = attn_operands(2, 200, 4, 2, 48, 64, dtype, "token", seed=14)
    clean = linear_attention_fn(q, k, v, g)
    mag, _ = recurrence(*(t.double().abs() for t in (q, k, v)), g.double(), 1.0, torch.zeros(2, 4, 48, 64, dtype=torch.float64, device="cuda"))
    bound = 2 * ((200 / 16 + 200) * 2.0 ** -23 + 3 * ATTN_HALF[dtype]) * mag + 2 * TINY[dtype]
    for t in (0, 37, 150, 199):
        x = v.clone()
        x[0, t, 1, 5] = value
        o = linear_attention_fn(q, k, x, g)
        hit = torch.zeros_like(o, dtype=torch.bool)
        hit[0, t:, 1, 5] = True
        assert not bool(torch.isfinite(o[0, t, 1, 5]))
        within("values", o[~hit], clean[~hit].double(), bound[~hit])
        x = k.clone()
        x[0, t, 1, 5] = value
        o = linear_attention_fn(q, x, v, g)
        hit = torch.zeros_like(o, dtype=torch.bool)
        hit[0, t:, 2:] = True
        within("keys", o[~hit], clean[~hit].double(), bound[~hit])
        x = q.clone()
        x[0, t, 1, 5] = value
        o = linear_attention_fn(x, k, v, g)
        hit = torch.zeros_like(o, dtype=torch.bool)
        hit[0, t, 2:] = True
        within("queries", o[~hit], clean[~hit].double(), bound[~hit])


# ------------------------------------------------------------------------------------------------ calls that were answered wrongly


def test_model_embedding_is_a_module():
    """The model calls its embedding as a module: hooks on it run, and a module put in its place is the one that is called."""
    from lrnnx_b200.lm import MambaLMHeadModel
    torch.manual_seed(0)
    m = MambaLMHeadModel(32, 1, 100, device="cuda")
    ids = torch.randint(0, 100, (2, 9), device="cuda")
    seen = []
    handle = m.backbone.embedding.register_forward_hook(lambda module, args, out: seen.append(out.shape))
    want = m(ids)
    handle.remove()
    assert seen == [(2, 9, 32)] and isinstance(m.backbone.embedding, torch.nn.Embedding)
    plain = torch.nn.Embedding(100, 32, device="cuda")
    plain.weight = m.backbone.embedding.weight
    m.backbone.embedding = torch.nn.Sequential(plain, torch.nn.Identity())
    assert torch.equal(m(ids), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_with_any_stride(dtype):
    """The pitch of a single row, or of a single class, means nothing and may be zero."""
    from lrnnx_b200.ops import linear_cross_entropy, token_embedding
    h, w, labels = loss_operands(6, 40, 24, dtype)
    one = h[0].expand(6, 24)[:1]
    assert one.stride(0) == 0
    want = linear_cross_entropy(h[:1], w, labels[:1], reduction="none")
    assert torch.equal(linear_cross_entropy(one, w, labels[:1], reduction="none"), want)
    hg, wg = h[:1].clone().requires_grad_(), w[0].expand(5, 24)[:1].requires_grad_()
    loss = linear_cross_entropy(hg, wg, torch.zeros_like(labels[:1]))
    a = torch.autograd.grad(loss, (hg, wg))
    # the softmax of one class is one: three roundings of log-sums up to 8 in the loss, times values up to 4 in the gradients
    assert abs(float(loss.detach())) <= 3 * 2.0 ** -21 and all(float(x.float().abs().max()) <= 3 * 2.0 ** -19 for x in a)
    assert torch.equal(token_embedding(torch.zeros(3, dtype=torch.int64, device="cuda"), one.detach()), h[:1].expand(3, 24))


def test_second_derivatives_are_refused():
    """The gradients have no gradients of their own: asking for them is an error and not a silent zero."""
    from lrnnx_b200.ops import linear_attention_fn, linear_cross_entropy, token_embedding
    h, w, labels = loss_operands(6, 40, 24, torch.float32)
    q, k, v, g, _ = attn_operands(1, 5, 1, 1, 8, 8, torch.float32, "step")[0]
    ids = labels.clamp(0, 39)
    for make, x in ((lambda x: linear_cross_entropy(x, w, labels), h), (lambda x: token_embedding(ids, x).square().sum(), w),
                    (lambda x: linear_attention_fn(x, k, v, g).square().sum(), q)):
        x = x.detach().clone().requires_grad_()
        dx, = torch.autograd.grad(make(x), x, create_graph=True)
        assert torch.equal(dx, torch.autograd.grad(make(x), x)[0])
        with pytest.raises(RuntimeError, match="differentiated again"):
            (dx.sum() + x.sum()).backward()
