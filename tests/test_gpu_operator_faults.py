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


@pytest.mark.parametrize("spread,classes,features", [(1.0, 50280, 64), (4.0, 50280, 48), (2.0, 131072, 16), (0.5, 300, 64)])
def test_float16_gradients_keep_small_probabilities(spread, classes, features):
    """Row weights from 1e-4 to 1 of the largest and probabilities around 1 / classes.  dz is rounded to half a step of itself, at
    least 2^-25 in units of a 2^15th of the largest row weight: 2^-40 of it, where a row's own weight is 1e-4 = 2^-13.3 of it.  The
    other terms are those of any gradient; weights are positive on average, so that the softmax's part of a row's gradient does not cancel."""
    from lrnnx_b200.ops import linear_cross_entropy
    rows, u = 96, 2.0 ** -11
    h, w, labels = loss_operands(rows, classes, features, torch.float16, spread=spread)
    w = (w.float() + 0.25).to(torch.float16)
    up = 1024 * 10.0 ** -torch.linspace(0, 4, rows, device="cuda")
    hh, ww = h.detach().requires_grad_(), w.detach().requires_grad_()
    got = torch.autograd.grad(linear_cross_entropy(hh, ww, labels, reduction="none"), (hh, ww), up)
    ref = reference(h, w, labels, up)
    e = ref["p_err"] + u * ref["dz"].abs() + 2.0 ** -40 * ref["unit"]
    for name, x, err, mag, n in (("dh", got[0], e @ w.double().abs(), ref["dz"].abs() @ w.double().abs(), classes),
                                 ("dw", got[1], e.t() @ h.double().abs(), ref["dz"].abs().t() @ h.double().abs(), rows)):
        within(name, x, ref[name], err + (n / 16 + 8) * 2.0 ** -23 * mag + u * ref[name].abs() + 2.0 ** -25)


def test_float16_gradients_at_the_largest_scale():
    """A certain row's dz is at most 2 float16 steps over its weight, 2^15 units: no overflow, and none where the upstream gradient is huge."""
    from lrnnx_b200.ops import linear_cross_entropy
    h, w = torch.full((4, 8), 8.0, dtype=torch.float16, device="cuda"), torch.zeros(5, 8, dtype=torch.float16, device="cuda")
    w[0], w[1] = 8.0, -8.0                               # logits 512 and -512: the first class for certain
    labels = torch.tensor([0, 1, 2, 0], device="cuda")
    for up in (1.0, 2.0 ** 12, 2.0 ** -12):
        hh, ww = h.clone().requires_grad_(), w.clone().requires_grad_()
        dh, dw = torch.autograd.grad(linear_cross_entropy(hh, ww, labels, reduction="none"), (hh, ww), torch.full((4,), up, device="cuda"))
        want = torch.zeros(4, 8, device="cuda")
        want[1], want[2] = 16.0 * up, 8.0 * up           # W[0] - W[label]
        assert torch.equal(dh.float(), want.half().float())
        want = torch.zeros(5, 8, device="cuda")
        want[0], want[1], want[2] = 16.0 * up, -8.0 * up, -8.0 * up
        assert torch.equal(dw.float(), want.half().float())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_row_weight_that_is_not_finite_stays_in_its_row(value, dtype):
    """An upstream gradient that overflowed in one row leaves the other rows' hidden gradients as they are."""
    from lrnnx_b200.ops import linear_cross_entropy
    h, w, labels = loss_operands(40, 500, 64, dtype)
    labels[7] = 3
    up = 64 * (1 + torch.arange(40, device="cuda") % 7).float()
    rows = torch.arange(40, device="cuda") != 7
    clean, = torch.autograd.grad(linear_cross_entropy(h.requires_grad_(), w, labels, reduction="none"), h, up)
    up[7] = value
    got, = torch.autograd.grad(linear_cross_entropy(h, w, labels, reduction="none"), h, up)
    assert torch.equal(got[rows], clean[rows]) and not bool(torch.isfinite(got[7]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("features", [520, 1032, 1536, 8192])
def test_long_contractions_are_not_one_chain(features, dtype):
    """Every product is positive and the labels' class has none, so that what the tensor core truncates (2^-23 of the running sum at each 16
    features) adds up to one side in the log-sum-exp alone.  Chains hold 512 features (float32, with 8 steps' worth for the
    five small products) or 1024, and their sums are rounded."""
    from lrnnx_b200.ops import linear_cross_entropy
    gen = torch.Generator().manual_seed(features)
    h = torch.randn(150, features, generator=gen).abs().to(dtype).cuda()
    w = (torch.randn(600, features, generator=gen).abs() * (30 / (0.64 * features))).to(dtype).cuda()
    w[0] = 0
    labels = torch.zeros(150, dtype=torch.int64, device="cuda")
    hh, ww = h.requires_grad_(), w.requires_grad_()
    up = torch.full((150,), 4.0, device="cuda")
    loss = linear_cross_entropy(hh, ww, labels, reduction="none")
    ref = reference(h.detach(), w.detach(), labels, up)
    chain = 512 if dtype == torch.float32 else 1024
    z = (h.detach().double() @ w.detach().double().t()).amax(1)
    Z = z * (min(features, chain) / 16 + 8 + features // chain + 1) * 2.0 ** -23
    assert bool(((loss.detach().double() - ref["loss"]).abs() <= Z + 2.0 ** -21 * (1 + ref["lse"])).all())
    check(torch.autograd.grad(loss, (hh, ww), up), ref, h.detach(), w.detach(), dtype)


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


def test_step_refuses_a_state_that_shares_memory():
    """A broadcast state would be read and written by several blocks at once."""
    from lrnnx_b200.ops import linear_attention_step
    (q, k, v, g, _), _, _ = attn_operands(3, 1, 4, 2, 16, 8, torch.float32, "token")
    ops = [x[:, 0] for x in (q, k, v, g)]
    one = torch.zeros(1, 4, 16, 8, device="cuda")
    for state in (one.expand(3, -1, -1, -1), torch.zeros(3, 1, 16, 8, device="cuda").expand(-1, 4, -1, -1), torch.zeros(3, 4, 1, 8, device="cuda").expand(-1, -1, 16, -1)):
        with pytest.raises(RuntimeError, match="share memory"):
            linear_attention_step(state, *ops)
    out = linear_attention_step(one.expand(1, 4, 16, 8), *[x[:1] for x in ops])            # a batch of one has no pitch to speak of
    assert out.shape == (1, 4, 8) and bool(one.any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,n,heads,groups,dk,dv,decay", [(2, 1500, 2, 1, 64, 48, "token"), (1, 2048, 2, 2, 128, 64, "token"), (1, 1500, 2, 2, 64, 64, "strong"),
                                                          (2, 600, 3, 1, 40, 32, "strong")])
def test_decay_gradients_keep_32_bits(b, n, heads, groups, dk, dv, decay, dtype):
    """A decay's gradient is a sum over pairs of steps across it.  The 2-norm of its error against the root of the sums of the pairs' squares,
    which the recurrence of squared operands and doubled decays gives: a pair's product is off by its operands' split (2^-22), the decays'
    exponentials (2^-22) and the truncations of at most 16 partial sums on its way (2^-20), independent of one another: 2^-19 in all.  A
    gradient from sums of q dq - k dk along the sequence has the error of those sums, which with strong decays are many times the pairs'."""
    from lrnnx_b200.ops import linear_attention_fn
    ops, dout, dlast = attn_operands(b, n, heads, groups, dk, dv, dtype, "token", seed=31)
    if decay == "strong":
        ops[3] = torch.full_like(ops[3], -3.0)
    want = with_gradients(ops, 1.0, dout, dlast)[5]
    square = lambda x: x.double().square()  # noqa: E731
    pairs = with_gradients([square(x) for x in ops[:3]] + [2 * ops[3].double(), square(ops[4])], 1.0, square(dout), square(dlast))[5].sqrt()
    leaves = [x.detach().requires_grad_() for x in ops]
    o, last = linear_attention_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
    got, = torch.autograd.grad([o, last], leaves[3:4], [dout, dlast])
    assert float((got.double() - want).norm()) <= 2.0 ** -19 * float(pairs.norm())


# ------------------------------------------------------------------------------------------------ waits


@pytest.mark.parametrize("dtype", DTYPES)
def test_lanes_meet_before_accumulators_are_read(dtype):
    """Sizes at which the lanes of a warp part right before an accumulator is read: columns that end inside 32, rows that cannot leave as a
    tile, several chunks and chains; results as for any size, the same twice, and no bounded wait ran out."""
    from lrnnx_b200 import _lib
    from lrnnx_b200.ops import linear_attention_fn, linear_cross_entropy
    h, w, labels = loss_operands(700, 1301, 509, dtype)
    hh, ww = h.detach().requires_grad_(), w.detach().requires_grad_()
    up = torch.tensor(700.0, device="cuda")
    runs = [torch.autograd.grad(linear_cross_entropy(hh, ww, labels), (hh, ww), up) for _ in range(2)]
    counted = int((labels != -100).sum())
    check(runs[0], reference(h, w, labels, torch.full((700,), 700 / counted, device="cuda", dtype=torch.float64)), h, w, dtype)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    for dk, dv in ((33, 81), (121, 99)):
        ops, dout, dlast = attn_operands(2, 391, 3, 1, dk, dv, dtype, "token", seed=21)
        want = with_gradients(ops, 1.0, dout, dlast)
        mag = with_gradients([x.abs() for x in ops[:3]] + [ops[3], ops[4].abs()], 1.0, dout.abs(), dlast.abs())
        runs = []
        for _ in range(2):
            leaves = [x.detach().requires_grad_() for x in ops]
            o, last = linear_attention_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
            runs.append([o.detach(), last.detach(), *torch.autograd.grad([o, last], leaves, [dout, dlast])])
        assert all(torch.equal(a, b) for a, b in zip(*runs))
        F, u = (391 / 16 + 200) * 2.0 ** -23, ATTN_HALF[dtype]
        for i in (0, 2, 3, 4):
            within(str(i), runs[0][i], want[i], (F + 2 * u) * mag[i] + u * want[i].abs() + TINY[dtype])
        for i in (1, 6):
            within(str(i), runs[0][i], want[i], F * mag[i])
    torch.cuda.synchronize()
    assert _lib.lib().b200_device_status() == 0


def test_waits_that_end_in_time_leave_no_status():
    """A wait that ran out ends its block whole (all threads read the same decision) and sets the status word, which ordinary calls of every
    path leave at zero: TMA or not, segments or not, with and without the gradient of the decays."""
    from lrnnx_b200 import _lib
    from lrnnx_b200.ops import linear_attention_fn
    for b, n, heads, dk, dv, pad in ((1, 4000, 1, 64, 64, 0), (1, 4000, 1, 128, 128, 3), (8, 140, 24, 128, 64, 0), (2, 129, 2, 50, 30, 1)):
        (q, k, v, g, s0), dout, dlast = attn_operands(b, n, heads, heads, dk, dv, torch.bfloat16, "token", seed=22)
        if pad:
            q, k, v = (torch.nn.functional.pad(x, (pad, pad))[..., pad:-pad] for x in (q, k, v))
        for with_g in (False, True):
            leaves = [x.detach().requires_grad_(i != 3 or with_g) for i, x in enumerate((q, k, v, g, s0))]
            o, last = linear_attention_fn(*leaves[:4], initial_state=leaves[4], return_last_state=True)
            grads = torch.autograd.grad([o, last], [x for x in leaves if x.requires_grad], [dout, dlast])
            assert all(bool(torch.isfinite(x).all()) for x in (o, last, *grads))
    torch.cuda.synchronize()
    assert _lib.lib().b200_device_status() == 0


# ------------------------------------------------------------------------------------------------ derivatives


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(grad):
    """A forward-mode tangent on any operand is an error, never dropped, whether gradients are recorded or not."""
    import torch.autograd.forward_ad as fw
    from lrnnx_b200.lm import MambaLMHeadModel
    from lrnnx_b200.ops import linear_attention_fn, linear_cross_entropy, token_embedding
    h, w, labels = loss_operands(6, 40, 24, torch.float32)
    ids = labels.clamp(0, 39)
    attn, _, _ = attn_operands(1, 5, 2, 1, 8, 8, torch.float32, "token")
    calls = [(lambda x: token_embedding(ids, x), w), (lambda x: linear_cross_entropy(x, w, labels), h), (lambda x: linear_cross_entropy(h, x, labels), w)]
    for i in range(5):
        calls.append((lambda x, i=i: linear_attention_fn(*[x if j == i else t for j, t in enumerate(attn[:4])], initial_state=x if i == 4 else attn[4]), attn[i]))
    model = MambaLMHeadModel(32, 1, 40, device="cuda")
    calls.append((lambda x: torch.func.functional_call(model, {"backbone.embedding.weight": x}, (ids[None],)), model.lm_head.weight.detach()))
    with torch.set_grad_enabled(grad), fw.dual_level():
        for call, x in calls:
            call(x)
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
                call(fw.make_dual(x, torch.ones_like(x)))
    # on the upstream gradient
    x = w.clone().requires_grad_()
    out = token_embedding(ids, x)
    with fw.dual_level():
        dout = torch.ones_like(out)
        torch.autograd.grad(out, x, dout, retain_graph=True)
        with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward"):
            torch.autograd.grad(out, x, fw.make_dual(dout, dout))


def test_transforms_are_refused():
    """torch.func's transforms of the operators are errors."""
    from lrnnx_b200.ops import linear_attention_fn, linear_cross_entropy, token_embedding
    h, w, labels = loss_operands(6, 40, 24, torch.float32)
    ids = labels.clamp(0, 39)
    q, k, v, g, _ = attn_operands(1, 5, 2, 1, 8, 8, torch.float32, "token")[0]
    for call, x in ((lambda x: token_embedding(ids, x).sum(), w), (lambda x: linear_cross_entropy(x, w, labels), h), (lambda x: linear_attention_fn(x, k, v, g).sum(), q)):
        for transform in (lambda: torch.func.grad(call)(x), lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.vmap(call)(torch.stack([x, x]))):
            with pytest.raises((NotImplementedError, RuntimeError)):
                transform()
    with pytest.raises(RuntimeError):
        torch.vmap(lambda i: token_embedding(i, w))(torch.stack([ids, ids]))


def test_second_derivatives_of_copied_operands_are_refused():
    """As for operands that are read in place: transposed ones, ones with other strides and more dimensions, one alone that requires a gradient."""
    from lrnnx_b200.ops import linear_attention_fn, linear_cross_entropy, token_embedding
    h, w, labels = loss_operands(6, 40, 24, torch.float32)
    attn, _, _ = attn_operands(1, 5, 2, 1, 8, 8, torch.float32, "token")
    turned = lambda x: x.transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731
    calls = [(lambda x: linear_cross_entropy(turned(x), w, labels), h), (lambda x: linear_cross_entropy(h, turned(x), labels), w),
             (lambda x: linear_cross_entropy(x.view(2, 3, 24), w, labels.view(2, 3)), h), (lambda x: linear_cross_entropy(turned(x.view(2, 3, 24)), w, labels.view(2, 3)), h),
             (lambda x: linear_cross_entropy(x[0].expand(6, 24)[:1], w, labels[:1].clamp(min=0)), h), (lambda x: token_embedding(labels.clamp(0, 39), turned(x)).square().sum(), w)]
    for i in range(5):
        calls.append((lambda x, i=i: linear_attention_fn(*[(turned(x) if i != 3 else x) if j == i else t for j, t in enumerate(attn[:4])],
                                                         initial_state=turned(x) if i == 4 else attn[4]).square().sum(), attn[i]))
    for call, x in calls:
        x = x.detach().clone().requires_grad_()
        dx, = torch.autograd.grad(call(x), x, create_graph=True)
        assert torch.equal(dx, torch.autograd.grad(call(x), x)[0]) and dx.requires_grad
        with pytest.raises(RuntimeError, match="differentiated again"):
            (dx.sum() + x.sum()).backward()


# ------------------------------------------------------------------------------------------------ the model


def _model(dtype, vocab=120):
    from lrnnx_b200.lm import MambaLMHeadModel
    torch.manual_seed(0)
    model = MambaLMHeadModel(32, 1, vocab, device="cuda", dtype=dtype)
    ids = torch.randint(0, vocab, (2, 19), device="cuda")
    labels = ids.roll(-1, 1)
    labels[0, 3:6], labels[1, 7] = -100, vocab + 5
    return model, ids, labels


def _of_logits(logits, labels, reduction):
    """The definition in float64."""
    z, y = logits.double().flatten(0, -2), labels.flatten()
    on = (y >= 0) & (y < z.shape[1])
    rows = torch.where(on, torch.logsumexp(z, 1) - z.gather(1, y.clamp(0, z.shape[1] - 1).unsqueeze(1)).squeeze(1), 0.0)
    return rows.view(labels.shape) if reduction == "none" else rows.sum() / (int((y != -100).sum()) if reduction == "mean" else 1)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("head", ["bias", "adapter", "hook", "pre_hook", "instance"])
def test_model_loss_calls_its_head(head, reduction):
    """``loss`` is the loss of ``model(ids)`` whatever module the head is: value and gradients, float32.  Logits are below 2 and losses near log 120, each
    with a few float32 roundings (2^-24) of 120 terms; the sum has 38 rows."""
    model, ids, labels = _model(torch.float32)
    weight = model.lm_head.weight
    if head == "bias":
        model.lm_head = torch.nn.Linear(32, 120, device="cuda")
        model.lm_head.weight = weight
    elif head == "adapter":
        model.lm_head = torch.nn.Sequential(torch.nn.Linear(32, 32, device="cuda"), model.lm_head)
    elif head == "hook":
        model.lm_head.register_forward_hook(lambda module, args, out: 3.0 * out + 1.0)
    elif head == "pre_hook":
        model.lm_head.register_forward_pre_hook(lambda module, args: (2.0 * args[0],))
    else:
        model.lm_head.forward = lambda x: torch.nn.functional.linear(x, weight) * 0.5
    params = list(model.parameters())
    want = _of_logits(model(ids), labels, reduction)
    got = model.loss(ids, labels, reduction=reduction)
    assert got.dtype == torch.float32 and got.shape == want.shape
    rows = 38 if reduction == "sum" else 1
    assert bool(((got.double() - want).abs() <= rows * 120 * 2.0 ** -22).all())
    for a, b in zip(torch.autograd.grad(got.sum(), params), torch.autograd.grad(want.sum(), params)):
        assert float((a - b).norm()) <= 2e-5 * float(b.norm()) + 1e-12


def test_model_loss_goes_through_forward():
    """What is hung on the model's own call sees the loss too, as a wrapper that calls ``forward`` does."""
    model, ids, labels = _model(torch.float32)
    seen = []
    model.register_forward_hook(lambda module, args, out: seen.append(out.shape))
    a, b = model.loss(ids, labels), model(ids, labels=labels)
    assert torch.equal(a, b) and seen == [(), ()]
    assert model(ids).shape == (2, 19, 120) and model.loss(ids, labels, reduction="none").shape == (2, 19)
    with pytest.raises(RuntimeError):
        model.loss(ids, labels[:, :-1])
    with pytest.raises(RuntimeError):
        model.loss(ids, labels, reduction="max")
    model.lm_head = torch.nn.Linear(32, 120, device="cuda")
    with pytest.raises(RuntimeError):
        model.loss(ids, labels[:, :-1])
    with pytest.raises(RuntimeError):
        model.loss(ids, labels, reduction="max")


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_model_loss_under_autocast(reduction):
    """Float32 weights under autocast leave hidden states of another type than the head's weight, which the model's call takes and its loss
    has to as well.  Logits below 2 are bfloat16, half a step 2^-8 of a value: a row's loss is off by two of them at most, with 38 rows in a sum."""
    model, ids, labels = _model(torch.float32)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):      # (the mixer's backward pass wants one type)
        logits = model(ids)
        got = model.loss(ids, labels, reduction=reduction)
    assert logits.dtype == torch.bfloat16 and got.dtype == torch.float32
    want = _of_logits(logits, labels, reduction)
    assert bool(((got.double() - want).abs() <= (38 if reduction == "sum" else 1) * 2 * 2.0 ** -8 * 2).all())


def test_calls_of_two_threads_at_once():
    """Threads with a stream each, which also look the driver's functions up for the first time together: the results of one thread alone."""
    import subprocess
    import sys
    from pathlib import Path
    here = Path(__file__).resolve().parent
    code = """
import sys, threading, torch
sys.path[:0] = [%r, %r]
from test_gpu_linear_attention import make as attn_operands
from test_gpu_linear_cross_entropy import make as loss_operands
from lrnnx_b200 import _lib
from lrnnx_b200.ops import linear_attention_fn, linear_attention_step, linear_cross_entropy, token_embedding
dt = torch.bfloat16
h, w, labels = loss_operands(300, 2000, 64, dt)
ids = labels.clamp(min=0)
(q, k, v, g, s0), dout, dlast = attn_operands(2, 700, 3, 1, 64, 64, dt, "token")
def run():
    L = [t.detach().requires_grad_() for t in (h, w, q, k, v, g)]
    loss, e, o = linear_cross_entropy(L[0], L[1], labels), token_embedding(ids, L[1]), linear_attention_fn(*L[2:])
    s = s0.clone()
    y = linear_attention_step(s, q[:, 0], k[:, 0], v[:, 0], g[:, 0])
    return [loss.detach(), o.detach(), y, s, *torch.autograd.grad([loss, e, o], L, [None, torch.ones_like(e), dout])]
got, start = [None] * 6, threading.Barrier(6)
def thread(i):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        start.wait()
        for _ in range(10):
            got[i] = run()
    stream.synchronize()
torch.cuda.synchronize()
threads = [threading.Thread(target=thread, args=(i,)) for i in range(6)]
for t in threads: t.start()
for t in threads: t.join()
want = run()
torch.cuda.synchronize()
assert all(len(r) == len(want) and all(torch.equal(a, b) for a, b in zip(r, want)) for r in got)
assert _lib.lib().b200_device_status() == 0
print("same")
""" % (str(here), str(here.parent))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr
