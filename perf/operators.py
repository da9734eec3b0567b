"""What a language model on this package runs at its two ends and in its mixer, and how each is measured.

kind     what                                                                   ranges
loss     softmax cross entropy of hidden @ weight^T without the logits          rows 1..16384, classes 64..131072, features 8..2048
embed    embedding lookup with a scale, its gradient by sorted tokens           tokens 1..65536, classes 16..131072, features 4..2048
attn     linear attention with a decay for each head over a sequence            batch 1..16, length 1..16384, head sizes 16..128
step     the same recurrence for one token, the state updated in place          batch 1..256, head sizes 16..128

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the package's operators."""
import math

import torch

own = False


def listed():
    return [
        # the training loss of the 130M model: 8 x 2048 tokens, vocabulary 50280, bfloat16
        dict(name="loss_lm_bf16", kind="loss", rows=16384, classes=50280, features=768, dtype="bfloat16", reduction="mean", grad=True),
        # a small float32 model on data and a vocabulary of no round size
        dict(name="loss_ragged_f32", kind="loss", rows=2031, classes=16411, features=509, dtype="float32", reduction="mean", grad=True),
        # scoring: the loss of every token of a few sequences under the 1.4B model's head, no gradient
        dict(name="loss_score_f16", kind="loss", rows=333, classes=50280, features=2048, dtype="float16", reduction="none", grad=False),
        # the embedding of the same training step, token frequencies as in text
        dict(name="embed_lm_bf16", kind="embed", tokens=16384, classes=50280, features=768, dtype="bfloat16", scaled=False, zipf=True, pad=False, grad=True),
        # the lookup of one decoding step, 64 sequences: the smallest call there is
        dict(name="embed_step_bf16", kind="embed", tokens=64, classes=50280, features=2048, dtype="bfloat16", scaled=False, zipf=True, pad=False, grad=False),
        # a character-sized vocabulary in float32 with a scale and a padding token: thousands of rows for each class
        dict(name="embed_ragged_f32", kind="embed", tokens=40007, classes=257, features=250, dtype="float32", scaled=True, zipf=False, pad=True, grad=True),
        # a layer in training at the 130M shape: 24 heads of 64, keys of 128 shared by all heads, decay from the input
        dict(name="attn_train_bf16", kind="attn", batch=8, length=2048, heads=24, groups=1, dk=128, dv=64, dtype="bfloat16", decay="token", resets=False,
             state=False, grad=True),
        # float32 training on lengths and heads of odd size, packed documents, a state carried in and out
        dict(name="attn_ragged_f32", kind="attn", batch=3, length=777, heads=6, groups=3, dk=48, dv=77, dtype="float32", decay="token", resets=True,
             state=True, grad=True),
        # the prompt of a long conversation: one sequence, a constant decay for each head, the state handed to decoding
        dict(name="attn_prefill_bf16", kind="attn", batch=1, length=16384, heads=16, groups=16, dk=128, dv=128, dtype="bfloat16", decay="head", resets=False,
             state=True, grad=False),
        # a short training call in float16, where launches count
        dict(name="attn_small_f16", kind="attn", batch=2, length=100, heads=8, groups=8, dk=64, dv=64, dtype="float16", decay="head", resets=False,
             state=False, grad=True),
        # decoding, 64 sequences in a pool of states, float32 states
        dict(name="step_64_bf16", kind="step", batch=64, heads=24, groups=1, dk=128, dv=64, dtype="bfloat16", state="float32", decay="token", pool=True),
        # decoding a single sequence
        dict(name="step_1_f32", kind="step", batch=1, heads=8, groups=8, dk=64, dv=64, dtype="float32", state="float32", decay="head", pool=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["loss", "loss", "embed", "attn", "attn", "step"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind == "loss":
        while True:
            c = dict(kind=kind, rows=_log(rng, 1, 16384), classes=_log(rng, 64, 131072), features=_log(rng, 8, 2048), dtype=dtype,
                     reduction=rng.choice(["mean", "mean", "sum", "none"]), grad=rng.random() < 0.7)
            if rng.random() < 0.5:
                c["features"] = max(8, c["features"] // 8 * 8)
            n = c["rows"] * c["classes"]
            if n <= 16384 * 50280 and n * c["features"] <= 16384 * 50280 * 768 // (8 if dtype == "float32" else 1):
                return c
    if kind == "embed":
        while True:
            c = dict(kind=kind, tokens=_log(rng, 1, 65536), classes=_log(rng, 16, 131072), features=_log(rng, 4, 2048), dtype=dtype,
                     scaled=rng.random() < 0.5, zipf=rng.random() < 0.5, pad=rng.random() < 0.3, grad=rng.random() < 0.7)
            if rng.random() < 0.5:
                c["features"] = max(8, c["features"] // 8 * 8)
            if (c["tokens"] + c["classes"]) * c["features"] <= 1 << 27:
                return c
    groups, per = rng.choice([1, 1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 8])
    size = lambda: rng.choice([16, 32, 64, 64, 128, 128, rng.randint(16, 128)])  # noqa: E731
    if kind == "step":
        while True:
            c = dict(kind=kind, batch=_log(rng, 1, 256), heads=groups * per, groups=groups, dk=size(), dv=size(), dtype=dtype,
                     state=rng.choice(["float32", "float32", dtype]), decay=rng.choice(["token", "head"]), pool=rng.random() < 0.5)
            if c["batch"] * c["heads"] * c["dk"] * c["dv"] <= 1 << 26:
                return c
    while True:
        c = dict(kind=kind, batch=_log(rng, 1, 16), length=_log(rng, 1, 16384), heads=groups * per, groups=groups, dk=size(), dv=size(), dtype=dtype,
                 decay=rng.choice(["token", "token", "head"]), resets=False, state=rng.random() < 0.5, grad=rng.random() < 0.6)
        c["resets"] = c["decay"] == "token" and rng.random() < 0.4
        if rng.random() < 0.5:
            c["length"] = max(1, c["length"] // 64 * 64)
        if c["batch"] * c["length"] * c["heads"] * (c["dk"] + c["dv"]) <= 16384 * 24 * 192:
            return c


# -------------------------------------------------------------------------------------------- inputs


def _prepare_loss(c, g, dt):
    n, v, d = c["rows"], c["classes"], c["features"]
    h = torch.randn(n, d, generator=g, device="cuda", dtype=dt)                                    # behind the last norm
    w = (torch.randn(v, d, generator=g, device="cuda") * (2 / math.sqrt(d))).to(dt)                # logits of spread 2
    labels = torch.randint(v, (n,), generator=g, device="cuda")
    labels[torch.rand(n, generator=g, device="cuda") < 1 / 16] = -100                              # prompts and ends of documents
    s = {"h": h.requires_grad_(c["grad"]), "w": w.requires_grad_(c["grad"]), "labels": labels}
    if c["reduction"] == "none":
        s["dloss"] = torch.rand(n, generator=g, device="cuda") + 0.5                               # a weight for each token
    else:
        # float16 is trained with a scaled loss
        s["dloss"] = torch.tensor(float(n) if c["dtype"] == "float16" and c["reduction"] == "mean" else 1.0, device="cuda")
    return s


def _prepare_embed(c, g, dt):
    n, v, d = c["tokens"], c["classes"], c["features"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(v + 1)) - 1 if c["zipf"] else u * v).long().clamp(0, v - 1)      # the r-th token with frequency 1 / r, or all alike
    s = {"ids": ids, "w": torch.randn(v, d, generator=g, device="cuda", dtype=dt).requires_grad_(c["grad"])}
    if c["grad"]:
        s["dout"] = torch.randn(n, d, generator=g, device="cuda", dtype=dt)
    return s


def _decay(c, g, shape):
    """Log decays: of a head, 1 - 2^-5 .. 1 - 2^-12 over the heads; of a token, step size times rate, between -1.6 and -0.001."""
    if c["decay"] == "head":
        return torch.log1p(-torch.exp2(-5 - 7 * torch.arange(c["heads"], device="cuda") / max(1, c["heads"] - 1)))
    d = -torch.exp(torch.rand(shape, generator=g, device="cuda") * math.log(1600.0)) * 1e-3
    if c.get("resets"):                                                                            # a new document starts with an empty state
        d[torch.rand(shape[:-1], generator=g, device="cuda") < 1 / 200] = -math.inf
    return d


def _prepare_attn(c, g, dt):
    b, n, h, r, dk, dv = (c[k] for k in ("batch", "length", "heads", "groups", "dk", "dv"))
    r_ = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = {"q": r_(b, n, r, dk).to(dt), "k": (r_(b, n, r, dk) / math.sqrt(dk)).to(dt), "v": r_(b, n, h, dv).to(dt), "g": _decay(c, g, (b, n, h)),
         "s0": r_(b, h, dk, dv) if c["state"] else None}
    if c["grad"]:
        for k in ("q", "k", "v", "g", "s0"):
            if s[k] is not None:
                s[k].requires_grad_()
        s["dout"] = r_(b, n, h, dv).to(dt)
        s["dlast"] = r_(b, h, dk, dv) if c["state"] else None
    return s


def _prepare_step(c, g, dt):
    b, h, r, dk, dv = (c[k] for k in ("batch", "heads", "groups", "dk", "dv"))
    r_ = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    slots = 2 * b if c["pool"] else b
    at = torch.randperm(slots, generator=g, device="cuda")[:b].to(torch.int32) if c["pool"] else None
    return {"state": r_(slots, h, dk, dv).to(_dt(c["state"])), "at": at, "q": r_(b, r, dk).to(dt), "k": (r_(b, r, dk) / math.sqrt(dk)).to(dt),
            "v": r_(b, h, dv).to(dt), "g": _decay(c, g, (b, h))}


def _dt(name):
    return getattr(torch, name)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"case": case, **globals()["_prepare_" + case["kind"]](case, g, _dt(case["dtype"]))}


# --------------------------------------------------------------------------------------- plain forms


def _scale(c):
    return math.sqrt(c["features"]) if c["kind"] == "embed" and c["scaled"] else 1.0 if c["kind"] == "embed" else c["dk"] ** -0.5


def _plain_loss(s):
    c, labels = s["case"], s["labels"]
    h, w = s["h"].float(), s["w"].float()
    z = h @ w.t()
    m = z.amax(1, keepdim=True)
    p = torch.exp(z - m)
    total = p.sum(1, keepdim=True)
    valid = labels != -100
    at = labels.clamp(min=0).unsqueeze(1)
    loss = torch.where(valid, (torch.log(total) + m - z.gather(1, at)).squeeze(1), 0)
    share = torch.ones_like(loss)
    if c["reduction"] == "mean":
        share = share / valid.sum().clamp(min=1)
    out = loss if c["reduction"] == "none" else (loss * share).sum()
    if not c["grad"]:
        return [out]
    del z
    p = p.div_(total)
    p.scatter_add_(1, at, torch.full_like(m, -1.0))
    p *= (torch.where(valid, share, 0) * s["dloss"]).unsqueeze(1)
    return [out, (p @ w).to(s["h"].dtype), (p.t() @ h).to(s["w"].dtype)]


def _plain_embed(s):
    c = s["case"]
    out = [(s["w"].detach()[s["ids"]].float() * _scale(c)).to(s["w"].dtype)]
    if c["grad"]:
        d = s["dout"].float() * _scale(c)
        if c["pad"]:
            d = torch.where((s["ids"] == 0).unsqueeze(1), 0, d)
        out.append(torch.zeros_like(s["w"], dtype=torch.float32).index_add_(0, s["ids"], d).to(s["w"].dtype))
    return out


def _chunked(q, k, v, g, s0, scale, chunk=64):
    """The recurrence in pieces: products inside a piece, and a triangular product over the pieces' states. All (batch, heads, length, ...), 32 bits; g in 64."""
    b, h, n, dk = q.shape
    pad = -n % chunk
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).unflatten(2, (-1, chunk)) for t in (q, k, v))
    G = torch.nn.functional.pad(g.clamp(min=-1e4), (0, pad)).unflatten(2, (-1, chunk)).cumsum(-1)
    low = torch.ones(chunk, chunk, dtype=torch.bool, device=q.device).tril()
    inside = (G.unsqueeze(-1) - G.unsqueeze(-2)).masked_fill(~low, -math.inf).exp().float()
    o = ((q @ k.transpose(-1, -2)) * inside) @ v
    last = G[..., -1:]
    own_state = (k * (last - G).exp().float().unsqueeze(-1)).transpose(-1, -2) @ v                 # what each piece adds
    P = torch.nn.functional.pad(last.squeeze(-1).cumsum(-1), (1, 0))                               # log decay up to each border
    m = P.shape[-1]
    before = torch.ones(m, m, dtype=torch.bool, device=q.device).tril(-1)[:, :-1]
    over = (P.unsqueeze(-1) - P[..., 1:].unsqueeze(-2)).masked_fill(~before, -math.inf).exp().float()
    S = (over @ own_state.flatten(-2)).unflatten(-1, own_state.shape[-2:])                         # at each border
    if s0 is not None:
        S = S + P.exp().float()[..., None, None] * s0.unsqueeze(2)
    o = o + (q * G.exp().float().unsqueeze(-1)) @ S[:, :, :-1]
    return scale * o.flatten(2, 3)[:, :, :n], S[:, :, -1]


def _plain_attn(s):
    c = s["case"]
    leaves = [t for t in (s["q"], s["k"], s["v"], s["g"], s["s0"]) if t is not None]
    with torch.set_grad_enabled(c["grad"]):
        wide = [t.detach().to(torch.float64 if t is s["g"] else torch.float32).requires_grad_(c["grad"]) for t in leaves]
        q, k, v, g = wide[:4]
        q, k = (t.repeat_interleave(c["heads"] // c["groups"], 2).transpose(1, 2) for t in (q, k))
        g = g.expand(c["batch"], c["length"], c["heads"]).transpose(1, 2)
        o, last = _chunked(q, k, v.transpose(1, 2), g, wide[4] if c["state"] else None, _scale(c))
        o = o.transpose(1, 2)
        out = [o.detach().to(s["v"].dtype)] + ([last.detach()] if c["state"] else [])
        if c["grad"]:
            ends, seeds = ([o, last], [s["dout"].float(), s["dlast"]]) if c["state"] else ([o], [s["dout"].float()])
            out += [d.to(t.dtype) for d, t in zip(torch.autograd.grad(ends, wide, seeds), leaves)]
    return out


def _plain_step(s):
    c, per = s["case"], s["case"]["heads"] // s["case"]["groups"]
    q, k = (s[x].float().repeat_interleave(per, 1) for x in "qk")
    g = s["g"].expand(c["batch"], c["heads"])
    at = s["at"].long() if c["pool"] else slice(None)
    S = s["state"][at].float() * torch.exp(g)[..., None, None] + k.unsqueeze(-1) * s["v"].float().unsqueeze(-2)
    s["state"][at] = S.to(s["state"].dtype)
    return [(_scale(c) * (q.unsqueeze(-1) * S).sum(-2)).to(s["v"].dtype), s["state"]]


# ------------------------------------------------------------------------------- the package's calls


def _own_loss(s):
    from lrnnx_b200.ops import linear_cross_entropy
    c = s["case"]
    loss = linear_cross_entropy(s["h"], s["w"], s["labels"], reduction=c["reduction"])
    return [loss.detach()] + (list(torch.autograd.grad(loss, (s["h"], s["w"]), s["dloss"])) if c["grad"] else [])


def _own_embed(s):
    from lrnnx_b200.ops import token_embedding
    c = s["case"]
    out = token_embedding(s["ids"], s["w"], scale=_scale(c), padding_idx=0 if c["pad"] else None)
    return [out.detach()] + (list(torch.autograd.grad(out, s["w"], s["dout"])) if c["grad"] else [])


def _own_attn(s):
    from lrnnx_b200.ops import linear_attention_fn
    c = s["case"]
    got = linear_attention_fn(s["q"], s["k"], s["v"], s["g"], scale=_scale(c), initial_state=s["s0"], return_last_state=c["state"])
    ends = list(got) if c["state"] else [got]
    out = [t.detach() for t in ends]
    if c["grad"]:
        leaves = [t for t in (s["q"], s["k"], s["v"], s["g"], s["s0"]) if t is not None]
        out += torch.autograd.grad(ends, leaves, [s["dout"], s["dlast"]][:len(ends)])
    return out


def _own_step(s):
    from lrnnx_b200.ops import linear_attention_step
    out = linear_attention_step(s["state"], s["q"], s["k"], s["v"], s["g"], scale=_scale(s["case"]), state_batch_indices=s["at"])
    return [out, s["state"]]


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


# ------------------------------------------------------------------------- what a pass has to move


def work(case):
    c, k = case, case["kind"]
    e = _dt(c["dtype"]).itemsize
    if k == "loss":
        n, v, d = c["rows"], c["classes"], c["features"]
        return {"bytes": e * (n + v) * d * (2 if c["grad"] else 1) + 12 * n, "flops": 2 * n * v * d * (3 if c["grad"] else 1)}
    if k == "embed":
        n, v, d = c["tokens"], c["classes"], c["features"]
        read = min(n, v) * d                                  # a row that several tokens share is read once
        return {"bytes": 8 * n + e * (read + n * d + ((n + v) * d if c["grad"] else 0)), "flops": n * d * (2 if c["grad"] else 1)}
    b, h, r, dk, dv = (c[x] for x in ("batch", "heads", "groups", "dk", "dv"))
    if k == "step":
        gb = 4 * (h if c["decay"] == "head" else b * h)
        return {"bytes": 2 * b * h * dk * dv * _dt(c["state"]).itemsize + e * b * (2 * r * dk + 2 * h * dv) + gb, "flops": 5 * b * h * dk * dv}
    t = b * c["length"]
    qkv, gb, st = e * t * (2 * r * dk + h * dv), 4 * (h if c["decay"] == "head" else t * h), 4 * b * h * dk * dv if c["state"] else 0
    fwd = qkv + gb + e * t * h * dv + 2 * st
    if not c["grad"]:
        return {"bytes": fwd, "flops": 4 * t * h * dk * dv}
    # backward: the operands and dout once more, a gradient for each operand
    return {"bytes": fwd + qkv + gb + e * t * h * dv + 2 * st + qkv + gb, "flops": 14 * t * h * dk * dv}


# ------------------------------------------------------------------ the definitions in 64 bits


def _exact_loss(c, s):
    h, w, labels, n = s["h"].detach().double(), s["w"].detach().double(), s["labels"], c["rows"]
    loss, dh, dw = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros_like(h), torch.zeros_like(w)
    counted = max(1, int((labels != -100).sum()))
    up = s["dloss"].double() / (counted if c["reduction"] == "mean" else 1)
    for a in range(0, n, 2048):
        rows = torch.arange(a, min(n, a + 2048), device="cuda")
        rows = rows[labels[rows] != -100]
        z = torch.log_softmax(h[rows] @ w.t(), dim=1)
        loss[rows] = -z[torch.arange(len(rows), device="cuda"), labels[rows]]
        if c["grad"]:
            dz = z.exp_()
            dz[torch.arange(len(rows), device="cuda"), labels[rows]] -= 1
            dz *= (up.expand(n)[rows]).unsqueeze(1)
            dh[rows] = dz @ w
            dw += dz.t() @ h[rows]
    out = loss if c["reduction"] == "none" else loss.sum() / (counted if c["reduction"] == "mean" else 1)
    return [out, dh, dw] if c["grad"] else [out]


def _exact_embed(c, s):
    ids, w = s["ids"], s["w"].detach().double()
    out = [w[ids] * _scale(c)]
    if c["grad"]:
        d = s["dout"].double() * _scale(c)
        order = torch.argsort(ids)
        ends = torch.bincount(ids, minlength=c["classes"]).cumsum(0)
        sums = torch.cat([torch.zeros(1, c["features"], dtype=torch.float64, device="cuda"), d[order].cumsum(0)])[ends]
        dw = sums - torch.cat([torch.zeros_like(sums[:1]), sums[:-1]])
        if c["pad"]:
            dw[0] = 0
        out.append(dw)
    return out


def _exact_attn(c, s):
    """Token by token."""
    b, n, h, per, scale = c["batch"], c["length"], c["heads"], c["heads"] // c["groups"], _scale(c)
    # time first: (length, batch, heads, size)
    q, k = (s[x].detach().double().transpose(0, 1).repeat_interleave(per, 2) for x in "qk")
    v = s["v"].detach().double().transpose(0, 1)
    g = s["g"].detach().double().expand(b, n, h).transpose(0, 1)
    a = g.exp()
    S = s["s0"].detach().double() if c["state"] else torch.zeros(b, h, c["dk"], c["dv"], dtype=torch.float64, device="cuda")
    o, dq = torch.empty_like(v), torch.empty_like(q)
    do = s["dout"].double().transpose(0, 1) if c["grad"] else None
    for t in range(n):
        S = S * a[t][..., None, None] + k[t].unsqueeze(-1) * v[t].unsqueeze(-2)
        o[t] = (q[t].unsqueeze(-2) @ S).squeeze(-2)
        if c["grad"]:
            dq[t] = (S @ do[t].unsqueeze(-1)).squeeze(-1)
    out = [scale * o.transpose(0, 1)] + ([S] if c["state"] else [])
    if not c["grad"]:
        return out
    dS = s["dlast"].double() if c["state"] else torch.zeros_like(S)
    end = (dS * S).sum((-1, -2))
    dk, dv = torch.empty_like(k), torch.empty_like(v)
    for t in range(n - 1, -1, -1):
        dS = dS + scale * q[t].unsqueeze(-1) * do[t].unsqueeze(-2)
        dk[t] = (dS @ v[t].unsqueeze(-1)).squeeze(-1)
        dv[t] = (k[t].unsqueeze(-2) @ dS).squeeze(-2)
        dS = dS * a[t][..., None, None]
    dq *= scale
    # a decay scales all that passes it: what later outputs and the last state take from before it
    dg = ((q * dq).sum(-1) - (k * dk).sum(-1)).flip(0).cumsum(0).flip(0) + end
    dg = torch.where(torch.isinf(g), 0.0, dg)
    fold = lambda t: t.unflatten(2, (c["groups"], per)).sum(3).transpose(0, 1)  # noqa: E731
    out += [fold(dq), fold(dk), dv.transpose(0, 1), dg.transpose(0, 1) if c["decay"] == "token" else dg.sum((0, 1))]
    return out + ([dS] if c["state"] else [])


def _exact_step(c, s):
    per = c["heads"] // c["groups"]
    q, k = (s[x].double().repeat_interleave(per, 1) for x in "qk")
    at = s["at"].long() if c["pool"] else torch.arange(c["batch"], device="cuda")
    S = torch.einsum("bhkv,bh->bhkv", s["state"].double()[at], torch.exp(s["g"].double().expand(c["batch"], c["heads"])))
    S += torch.einsum("bhk,bhv->bhkv", k, s["v"].double())
    state = s["state"].double()
    state[at] = S
    return [_scale(c) * torch.einsum("bhk,bhkv->bhv", q, S), state]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return globals()["_exact_" + case["kind"]](case, s)
