"""Linear attention with a decay for each head against the recurrence in float64, token by token.

Bounds, element by element.  M is the same result with every operand replaced by its magnitude (the sum of the
magnitudes of all products that enter it).  Float32 sums of chunks, states and splits: at most F = (length / 16 + 200) 2^-23 of M.  With
16-bit operands the scores and states that a result is made from may be rounded once to the type, u of M each, and
the result is rounded once.  States and decay gradients are float32 whatever the operands, and keep to F; a decay
gradient is a running sum of differences q . dq - k . dk, whose magnitudes are added up along the sequence."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}
DTYPES = list(HALF)


def recurrence(q, k, v, g, scale, s0):
    """The definition; q, k (b, l, groups, dk), v (b, l, h, dv), g (b, l, h) or (h,), all float64."""
    b, n, h, _ = v.shape
    per = h // q.shape[2]
    q, k = q.repeat_interleave(per, 2), k.repeat_interleave(per, 2)
    a = g.expand(b, n, h).exp()
    S, outs = s0, []
    for t in range(n):
        S = S * a[:, t, :, None, None] + k[:, t].unsqueeze(-1) * v[:, t].unsqueeze(-2)
        outs.append(scale * (q[:, t].unsqueeze(-2) @ S).squeeze(-2))
    return torch.stack(outs, 1), S


def with_gradients(ops, scale, dout, dlast):
    leaves = [t.double().requires_grad_() for t in ops]
    o, S = recurrence(*leaves[:4], scale, leaves[4])
    return [o.detach(), S.detach()] + list(torch.autograd.grad([o, S], leaves, [dout.double(), dlast.double()]))


def make(b, n, heads, groups, dk, dv, dtype, decay, seed=0):
    g_ = torch.Generator().manual_seed(seed * 7919 + b + n * 3 + heads * 5 + dk * 11 + dv * 13)
    r = lambda *s: torch.randn(*s, generator=g_)  # noqa: E731
    q, k, v = r(b, n, groups, dk).to(dtype), (r(b, n, groups, dk) / math.sqrt(dk)).to(dtype), r(b, n, heads, dv).to(dtype)
    if decay == "head":
        g = torch.log1p(-torch.exp2(-1 - 6 * torch.arange(heads) / max(1, heads - 1)))
    else:
        g = -torch.exp(torch.rand(b, n, heads, generator=g_) * math.log(3000.0)) * 1e-3
        if decay == "resets":
            g[torch.rand(b, n, generator=g_) < 0.1] = -math.inf
            g[:, 0] = -math.inf
    return [t.cuda() for t in (q, k, v, g, r(b, heads, dk, dv))], r(b, n, heads, dv).to(dtype).cuda(), r(b, heads, dk, dv).cuda()


def within(name, got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (name, float((off / bound.clamp(min=1e-300)).max()))


SIZES = [(1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 16, 8), (1, 63, 2, 2, 16, 16), (2, 64, 4, 2, 64, 64), (1, 65, 3, 1, 33, 65), (2, 130, 2, 2, 128, 128), (1, 257, 6, 3, 48, 77),
         (3, 191, 4, 4, 128, 64), (1, 700, 1, 1, 20, 100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay", ["head", "token", "resets"])
@pytest.mark.parametrize("b,n,heads,groups,dk,dv", SIZES)
def test_forward_and_gradients(b, n, heads, groups, dk, dv, decay, dtype):
    from lrnnx_b200.ops import linear_attention_fn
    (q, k, v, g, s0), dout, dlast = make(b, n, heads, groups, dk, dv, dtype, decay)
    scale = 0.7
    want = with_gradients((q, k, v, g, s0), scale, dout, dlast)
    mag = with_gradients([t.abs() for t in (q, k, v)] + [g, s0.abs()], scale, dout.abs(), dlast.abs())
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, s0)]
    o, last = linear_attention_fn(*leaves[:4], scale=scale, initial_state=leaves[4], return_last_state=True)
    got = [o, last] + list(torch.autograd.grad([o, last], leaves, [dout, dlast]))
    F, u, tiny = (n / 16 + 200) * 2.0 ** -23, HALF[dtype], TINY[dtype]
    for name, i in (("o", 0), ("dq", 2), ("dk", 3), ("dv", 4)):
        assert got[i].dtype == dtype
        within(name, got[i], want[i], (F + 2 * u) * mag[i] + u * want[i].abs() + tiny)
    for name, i in (("last", 1), ("ds0", 6)):
        assert got[i].dtype == torch.float32
        within(name, got[i], want[i], F * mag[i])
    # magnitudes of the differences that a decay gradient adds up
    per = heads // groups
    qa, ka = (t.abs().double().repeat_interleave(per, 2) for t in (q, k))
    each = with_gradients([qa, ka, v.abs(), g, s0.abs()], scale, dout.abs(), dlast.abs())
    run = ((qa * each[2]).sum(-1) + (ka * each[3]).sum(-1)).flip(1).cumsum(1).flip(1) + (dlast.abs().double() * mag[1]).sum((-1, -2)).unsqueeze(1)
    if decay == "head":
        run = run.sum((0, 1))
    assert got[5].dtype == torch.float32 and bool(torch.isfinite(got[5]).all())
    within("dg", got[5], torch.nan_to_num(want[5]), F * run)
    if decay == "resets":
        assert torch.count_nonzero(got[5][g == -math.inf]) == 0


@pytest.mark.parametrize("dtype,state", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.float16, torch.float16)])
@pytest.mark.parametrize("b,heads,groups,dk,dv", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (2, 3, 1, 128, 128), (5, 2, 2, 33, 77), (64, 6, 1, 128, 64), (2, 2, 2, 16, 8)])
def test_step(b, heads, groups, dk, dv, dtype, state):
    """One step, on a state and on a pool with entries that have no slot.  Product and sum of a state element round at most
    three times (2^-24 each) and once to its type; the output adds dk of them in float32."""
    from lrnnx_b200.ops import linear_attention_step
    for pool in (False, True):
        for decay in ("head", "token"):
            (q, k, v, g, _), _, _ = make(b, 1, heads, groups, dk, dv, dtype, decay, seed=3)
            q, k, v = q[:, 0], k[:, 0], v[:, 0]
            g = g if decay == "head" else g[:, 0]
            slots = 2 * b + 1 if pool else b
            gen = torch.Generator().manual_seed(b)
            S = torch.randn(slots, heads, dk, dv, generator=gen).to(state).cuda()
            at = torch.randperm(slots, generator=gen)[:b].to(torch.int32).cuda() if pool else None
            rows = at.long() if pool else torch.arange(b, device="cuda")
            if pool and b > 1:
                at[1] = -1
            before = S.clone()
            per = heads // groups
            qd, kd = (t.double().repeat_interleave(per, 1) for t in (q, k))
            a = g.double().expand(b, heads).exp()[..., None, None]
            new = before[rows].double() * a + kd.unsqueeze(-1) * v.double().unsqueeze(-2)
            mag = before[rows].double().abs() * a + (kd.unsqueeze(-1) * v.double().unsqueeze(-2)).abs()
            out = linear_attention_step(S, q, k, v, g, scale=0.7, state_batch_indices=at)
            want = 0.7 * (qd.unsqueeze(-1) * new).sum(-2)
            out_mag = 0.7 * (qd.abs().unsqueeze(-1) * mag).sum(-2)
            u, us = HALF[dtype], HALF[state]
            live = torch.ones(b, dtype=torch.bool, device="cuda")
            if pool and b > 1:
                live[1] = False
                assert torch.count_nonzero(out[1]) == 0
            within("out", out[live], want[live], ((dk + 8) * 2.0 ** -23 * out_mag + u * want.abs() + TINY[dtype])[live])
            within("state", S[rows[live]], new[live], (2.0 ** -21 * mag + us * new.abs() + TINY[state])[live])
            others = torch.ones(slots, dtype=torch.bool, device="cuda")
            others[rows[live]] = False
            assert torch.equal(S[others], before[others])


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_steps_is_the_whole_sequence(dtype):
    """A prompt's last state handed to single steps gives what one call over the whole sequence gives."""
    from lrnnx_b200.ops import linear_attention_fn, linear_attention_step
    (q, k, v, g, _), _, _ = make(2, 150, 4, 2, 64, 48, dtype, "token", seed=5)
    whole, last = linear_attention_fn(q, k, v, g, return_last_state=True)
    out, state = linear_attention_fn(q[:, :100], k[:, :100], v[:, :100], g[:, :100], return_last_state=True)
    F, u = (150 / 16 + 200) * 2.0 ** -23, HALF[dtype]
    mag, state_mag = recurrence(*(t.double().abs() for t in (q, k, v)), g.double(), 1.0, torch.zeros(2, 4, 64, 48, dtype=torch.float64, device="cuda"))
    within("prompt", out, whole[:, :100].double(), 2 * (F + 3 * u) * mag[:, :100] + TINY[dtype])
    for t in range(100, 150):
        got = linear_attention_step(state, q[:, t], k[:, t], v[:, t], g[:, t])
        within("step", got, whole[:, t].double(), 2 * (F + 3 * u) * mag[:, t] + TINY[dtype])
    within("state", state, last.double(), 2 * F * state_mag)
