"""Routing of tokens to experts and preference losses: what is measured.

A case is a dict of plain values.  Its ``kind`` says which operator it runs:

* ``route``   — ``topk_routing``: the k experts of each token from its scores
  (router logits, or the rows of a transport plan), their weights, the tokens
  per expert and the balance loss; with the gradient of the scores in training;
* ``balance`` — ``balance_loss``: counts and loss of a given assignment, and the
  gradient of the scores;
* ``logp``    — ``sequence_logp``: log ratios of the answers from the logits,
  and the gradient of the logits in training;
* ``prefer``  — ``preference_loss``: the loss over pairs of log ratios or over a
  transport plan between two sets of them, and its gradients.

``own`` selects the framework's operators; without it ``run`` computes the
same from elementary operations in 32 bits (64 for long sums).
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_MOST_SCORES = 1 << 24  # elements of the largest score matrix that draw() makes
_MOST_LOGITS = 1 << 28  # and of the largest logits (the largest listed case has 2^30)
_MOST_PLAN = 1 << 24    # and of the largest plan


def _route(name, B, N, E, k, dtype, scoring="softmax", normalize=False, bias=False, valid=1.0, grad=True):
    return dict(name=name, kind="route", B=B, N=N, E=E, k=k, dtype=dtype, scoring=scoring, normalize=normalize,
                bias=bias, valid=valid, grad=grad)


def _balance(name, B, N, E, k, dtype, scoring="softmax", valid=1.0):
    return dict(name=name, kind="balance", B=B, N=N, E=E, k=k, dtype=dtype, scoring=scoring, valid=valid)


def _logp(name, B, S, V, dtype, tau=1.0, reduction="sum", ref="token", masked=True, grad=True):
    return dict(name=name, kind="logp", B=B, S=S, V=V, dtype=dtype, tau=tau, reduction=reduction, ref=ref,
                masked=masked, grad=grad)


def _prefer(name, P, Q, plan, loss_type="sigmoid", beta=0.1, smoothing=0.0):
    return dict(name=name, kind="prefer", P=P, Q=Q, plan=plan, loss_type=loss_type, beta=beta, smoothing=smoothing)


def listed():
    return [
        # Serving: the tokens of one decoding step of a few requests; latency.
        _route("route_decode", 1, 16, 256, 8, "bf16", "sigmoid", normalize=True, bias=True, grad=False),
        # Training with a few large experts, a batch of sequences.
        _route("route_coarse", 8, 4096, 16, 2, "bf16"),
        # Training with many small experts, fp32 router, balanced by a bias.
        _route("route_fine", 4, 16384, 256, 8, "fp32", "sigmoid", normalize=True, bias=True),
        # Routing over a Sinkhorn plan, an odd number of experts, padded batch.
        _route("route_plan", 3, 1999, 61, 3, "fp32", "plan", normalize=True, valid=0.7),
        # The loss of a small router on its own, few tokens.
        _balance("balance_small", 2, 300, 8, 2, "fp16"),
        # The loss over one long packed batch.
        _balance("balance_long", 1, 131072, 128, 6, "bf16"),
        # Scoring the last tokens of an answer, token by token; latency.
        _logp("logp_score", 1, 7, 32768, "bf16", reduction="none", ref="none", masked=False, grad=False),
        # Training on a batch of answers with masked prompts and padding.
        _logp("logp_train", 8, 1023, 32768, "bf16"),
        # Answers of a few tokens over an odd vocabulary, fp32, mean per token.
        _logp("logp_odd", 6, 129, 50021, "fp32", tau=0.7, reduction="mean", ref="sequence"),
        # Long answers over a large vocabulary: the largest call.
        _logp("logp_long", 4, 2048, 131072, "bf16"),
        # The loss of a batch of answer pairs; latency.
        _prefer("prefer_pairs", 64, 64, False, smoothing=0.1),
        # Two sets of answers coupled by a transport plan.
        _prefer("prefer_plan", 4096, 4096, True),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(["route", "route", "balance", "logp", "logp", "prefer"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if kind in ("route", "balance"):
        E = _log_uniform(rng, 4, 512)
        if rng.random() < 0.5:
            E = max(8, E // 8 * 8)
        B = rng.randint(1, 8)
        N = _log_uniform(rng, 1, min(65536, _MOST_SCORES // (B * E)))
        k = rng.randint(1, min(8, E))
        scoring = rng.choice(["softmax", "sigmoid", "plan"])
        valid = rng.choice([1.0, 1.0, 0.3, 0.8])
        if kind == "balance":
            return _balance("", B, N, E, k, "fp32" if scoring == "plan" else dtype, scoring, valid)
        return _route("", B, N, E, k, "fp32" if scoring == "plan" else dtype, scoring, rng.random() < 0.5,
                      scoring != "plan" and rng.random() < 0.5, valid, rng.random() < 0.8)
    if kind == "logp":
        V = _log_uniform(rng, 1000, 160000)
        if rng.random() < 0.5:
            V = V // 64 * 64 + 64
        B = rng.randint(1, 16)
        S = _log_uniform(rng, 1, max(1, min(4096, _MOST_LOGITS // (B * V))))
        reduction = rng.choice(["sum", "mean", "none"])
        # a token has no share of a sequence's reference
        ref = rng.choice(["token", "none"] if reduction == "none" else ["token", "sequence", "none"])
        return _logp("", B, S, V, dtype, rng.choice([1.0, 1.0, 0.6, 1.3]), reduction, ref, rng.random() < 0.7,
                     rng.random() < 0.8)
    P = _log_uniform(rng, 1, 8192)
    plan = rng.random() < 0.7
    Q = _log_uniform(rng, 1, min(8192, _MOST_PLAN // P)) if plan else P
    loss_type = rng.choice(["sigmoid", "hinge", "square"])
    return _prefer("", P, Q, plan, loss_type, rng.choice([0.05, 0.1, 0.5]),
                   rng.choice([0.0, 0.1]) if loss_type == "sigmoid" else 0.0)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")  # the CPU: to look at the forms only
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    make = dict(device=dev, generator=gen)
    c = dict(case)
    if c["kind"] in ("route", "balance"):
        return _prepare_scores(c, dev, make)
    if c["kind"] == "logp":
        return _prepare_logits(c, dev, make)
    return _prepare_ratios(c, dev, make)


def _prepare_scores(c, dev, make):
    B, N, E, k = c["B"], c["N"], c["E"], c["k"]
    # Router logits of unit order with experts that are liked more than others.
    scores = torch.randn(B, N, E, **make) + 0.5 * torch.randn(E, **make)
    experts = None
    if c["kind"] == "balance":
        noisy = scores + 0.5 * torch.randn(B, N, E, **make)
        experts = noisy.topk(k, dim=-1).indices.to(torch.int32)
    if c["scoring"] == "plan":
        # Rows of mass 1 / N, as a plan between N tokens and E experts has them.
        scores = torch.softmax(2.0 * scores, dim=-1) / N
    s = dict(case=c, scores=scores.to(_DTYPES[c["dtype"]]), experts=experts, bias=None, mask=None)
    if c.get("bias"):
        s["bias"] = 0.2 * torch.randn(E, **make)
    if c["valid"] < 1.0:
        s["mask"] = torch.rand(B, N, **make) < c["valid"]
    if c["kind"] == "route":
        s["grad_weights"] = torch.randn(B, N, k, **make)
    # the balance loss enters the training loss with a weight of its own
    s["grad_loss"] = 0.5 + torch.rand(B, **make)
    if c.get("grad", True):
        s["scores"].requires_grad_()
    return s


def _prepare_logits(c, dev, make):
    B, S, V = c["B"], c["S"], c["V"]
    dtype = _DTYPES[c["dtype"]]
    logits = torch.randn(B, S, V, dtype=dtype, **make).mul_(2.0)
    tokens = torch.randint(0, V, (B, S), **make)
    # The taken token's logit: from unlikely to nearly certain against the rest.
    taken = math.log(V) - 3.0 + 10.0 * torch.rand(B, S, **make)
    logits.scatter_(2, tokens.unsqueeze(2), taken.to(dtype).unsqueeze(2))
    s = dict(case=c, logits=logits, tokens=tokens, mask=None, ref=None)
    if c["masked"]:
        at = torch.arange(S, device=dev)
        prompt = (torch.rand(B, 1, **make) * 0.4 * S).long()
        end = ((0.5 + 0.5 * torch.rand(B, 1, **make)) * S).long() + 1
        s["mask"] = (at >= prompt) & (at < end)
    if c["ref"] != "none":
        # A reference model near this one: its log-probabilities to within about 0.5.
        rest = math.log(V) + 2.0 / c["tau"] ** 2  # the log of the sum over the other logits
        t = taken / c["tau"]
        ref = t - torch.logaddexp(t, torch.full_like(t, rest)) + 0.5 * torch.randn(B, S, **make)
        if c["ref"] == "sequence":
            held = ref if s["mask"] is None else ref * s["mask"]
            ref = held.sum(1)
            if c["reduction"] == "mean":
                n = torch.full_like(ref, S) if s["mask"] is None else s["mask"].sum(1)
                ref = ref / n.clamp(min=1)
        s["ref"] = ref
    s["grad"] = torch.randn(B, S, **make) if c["reduction"] == "none" else torch.randn(B, **make)
    if c["grad"]:
        s["logits"].requires_grad_()
    return s


def _prepare_ratios(c, dev, make):
    P, Q = c["P"], c["Q"]
    ratio = 4.0 * torch.randn(P + Q, **make)
    ratio[:P] += 2.0
    s = dict(case=c, ratio=ratio, plan=None, grad=torch.rand(P, **make) + 0.5)
    if c["plan"]:
        e = torch.exp(2.0 * torch.randn(P, Q, **make))
        s["plan"] = (e / e.sum(1, keepdim=True) / P).requires_grad_()
    s["ratio"].requires_grad_()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"route": _own_route, "balance": _own_balance, "logp": _own_logp, "prefer": _own_prefer}[kind](state)
    return {"route": _plain_route, "balance": _plain_balance, "logp": _plain_logp, "prefer": _plain_prefer}[kind](state)


def _own_route(s):
    import dot_amd

    c = s["case"]
    r = dot_amd.topk_routing(s["scores"], c["k"], scoring=c["scoring"], normalize=c["normalize"], bias=s["bias"],
                             mask=s["mask"])
    out = dict(weights=r.weights, experts=r.experts, counts=r.counts, balance_loss=r.balance_loss)
    if c["grad"]:
        (out["grad_scores"],) = torch.autograd.grad([r.weights, r.balance_loss], [s["scores"]],
                                                    [s["grad_weights"], s["grad_loss"]])
    return out


def _own_balance(s):
    import dot_amd

    r = dot_amd.balance_loss(s["scores"], s["experts"], scoring=s["case"]["scoring"], mask=s["mask"])
    (g,) = torch.autograd.grad([r.loss], [s["scores"]], [s["grad_loss"]])
    return dict(loss=r.loss, counts=r.counts, grad_scores=g)


def _own_logp(s):
    import dot_amd

    c = s["case"]
    out = dot_amd.sequence_logp(s["logits"], s["tokens"], ref_logp=s["ref"], mask=s["mask"], tau=c["tau"],
                                reduction=c["reduction"])
    if not c["grad"]:
        return dict(logp=out)
    (g,) = torch.autograd.grad([out], [s["logits"]], [s["grad"]])
    return dict(logp=out, grad_logits=g)


def _own_prefer(s):
    import dot_amd

    c = s["case"]
    loss = dot_amd.preference_loss(s["ratio"], plan=s["plan"], beta=c["beta"], loss_type=c["loss_type"],
                                   label_smoothing=c["smoothing"])
    leaves = [s["ratio"]] + ([s["plan"]] if c["plan"] else [])
    grads = torch.autograd.grad([loss], leaves, [s["grad"]])
    return dict(loss=loss, **dict(zip(("grad_ratio", "grad_plan"), grads)))


# --- the plain form ---------------------------------------------------------
def _masses(x, scoring):
    """(q, p, sum of q) of each row: q the expert's mass, p its share of the row."""
    if scoring == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        q = e / e.sum(-1, keepdim=True)
        return q, q, None
    q = 1.0 / (1.0 + torch.exp(-x)) if scoring == "sigmoid" else x
    total = q.sum(-1, keepdim=True)
    return q, q / total, total


def _plain_loss(p, experts, mask, k):
    """Counts, balance loss and d loss / d p of each row (without the loss's upstream gradient)."""
    B, N, E = p.shape
    taken = torch.zeros(B, N, E, dtype=torch.int32, device=p.device)
    taken.scatter_add_(2, experts.clamp(min=0).long(), (experts >= 0).to(torch.int32))
    if mask is not None:
        taken = taken * mask.unsqueeze(-1)
        p = p * mask.unsqueeze(-1)
        n = mask.sum(1, dtype=torch.float64).unsqueeze(-1)
    else:
        n = torch.full((B, 1), float(N), dtype=torch.float64, device=p.device)
    counts = taken.sum(1, dtype=torch.int32)
    n1 = n.clamp(min=1.0)
    share = counts.double() / (k * n1)
    loss = (E * (share * (p.sum(1, dtype=torch.float64) / n1)).sum(-1)).float()
    return counts, loss, (E * share / n1).float().unsqueeze(1)


def _scores_grad(s, q, p, total, h, spread):
    """Gradient of the scores: h = d L / d p, spread = d L / d q of the taken experts alone."""
    scoring = s["case"]["scoring"]
    back = h - (p * h).sum(-1, keepdim=True)
    if scoring == "softmax":
        g = p * back + spread
    else:
        g = back / total + spread
        if scoring == "sigmoid":
            g = g * (q * (1.0 - q))
    if s["mask"] is not None:
        g = torch.where(s["mask"].unsqueeze(-1), g, torch.zeros_like(g))
    return g.to(s["scores"].dtype)


def _plain_route(s):
    c = s["case"]
    k, scoring = c["k"], c["scoring"]
    x = s["scores"].detach().float()
    key = x if s["bias"] is None else x + s["bias"]
    experts = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :k]
    q, p, total = _masses(x, scoring)
    at = experts
    if c["normalize"] and scoring == "softmax":
        chosen = x.gather(-1, at)
        e = torch.exp(chosen - chosen.amax(-1, keepdim=True))
        weights = e / e.sum(-1, keepdim=True)
    else:
        weights = q.gather(-1, at)
        mass = weights.sum(-1, keepdim=True)
        if c["normalize"]:
            weights = weights / mass
    if s["mask"] is not None:
        weights = weights * s["mask"].unsqueeze(-1)
        experts = torch.where(s["mask"].unsqueeze(-1), experts, -torch.ones_like(experts))
    counts, loss, slope = _plain_loss(p, experts, s["mask"], k)
    out = dict(weights=weights, experts=experts.to(torch.int32), counts=counts, balance_loss=loss)
    if c["grad"]:
        dw = s["grad_weights"]
        h = (s["grad_loss"].view(-1, 1, 1) * slope).expand_as(p)
        if c["normalize"]:
            dw = dw - (weights * dw).sum(-1, keepdim=True)
            dw = weights * dw if scoring == "softmax" else dw / mass
            spread = torch.zeros_like(x).scatter(-1, at, dw)
        elif scoring == "softmax":
            h = h.scatter_add(-1, at, dw)
            spread = 0.0
        else:
            spread = torch.zeros_like(x).scatter(-1, at, dw)
        out["grad_scores"] = _scores_grad(s, q, p, total, h, spread)
    return out


def _plain_balance(s):
    c = s["case"]
    q, p, total = _masses(s["scores"].detach().float(), c["scoring"])
    counts, loss, slope = _plain_loss(p, s["experts"], s["mask"], c["k"])
    h = (s["grad_loss"].view(-1, 1, 1) * slope).expand_as(p)
    return dict(loss=loss, counts=counts, grad_scores=_scores_grad(s, q, p, total, h, 0.0))


def _plain_logp(s):
    c = s["case"]
    z = s["logits"].detach().float()
    if c["tau"] != 1.0:
        z = z / c["tau"]
    at = s["tokens"].unsqueeze(-1)
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    # the sum of many and the difference of two large numbers, in 64 bits
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    lp = ((z.gather(-1, at) - top).double() - torch.log(total)).squeeze(-1)
    ref, mask = s["ref"], s["mask"]
    if ref is not None and ref.dim() == 2:
        lp = lp - ref
    keep = torch.ones_like(lp) if mask is None else mask.double()
    lp = lp * keep
    weight = keep
    if c["reduction"] != "none":
        lp = lp.sum(1)
        if c["reduction"] == "mean":
            n = keep.sum(1, keepdim=True).clamp(min=1.0)
            lp = lp / n.squeeze(1)
            weight = keep / n
        if ref is not None and ref.dim() == 1:
            lp = lp - ref
    out = dict(logp=lp.float())
    if c["grad"]:
        g = s["grad"] if c["reduction"] == "none" else s["grad"].unsqueeze(1)
        coef = (g * weight / c["tau"]).float().unsqueeze(-1)
        grad = (e / total.float()).neg_()
        grad.scatter_add_(-1, at, torch.ones_like(coef))
        out["grad_logits"] = grad.mul_(coef).to(s["logits"].dtype)
    return out


def _plain_prefer(s):
    c = s["case"]
    P, beta, eps = c["P"], c["beta"], c["smoothing"]
    r = s["ratio"].detach()
    if c["plan"]:
        gap = r[:P].unsqueeze(1) - r[P:].unsqueeze(0)
    else:
        gap = r[:P] - r[P:]
    if c["loss_type"] == "sigmoid":
        d = beta * gap
        tail = torch.log1p(torch.exp(-d.abs()))
        f = (1.0 - eps) * (tail + (-d).clamp(min=0.0)) + eps * (tail + d.clamp(min=0.0))
        slope = beta * (1.0 / (1.0 + torch.exp(-d)) - (1.0 - eps))
    elif c["loss_type"] == "hinge":
        room = 1.0 - beta * gap.double()  # next to the kink in 64 bits
        f = room.clamp(min=0.0).float()
        slope = -beta * (room > 0).float()
    else:
        miss = gap - 0.5 / beta
        f = miss * miss
        slope = 2.0 * miss
    g = s["grad"]
    if not c["plan"]:
        return dict(loss=f, grad_ratio=torch.cat([g * slope, -g * slope]))
    plan = s["plan"].detach()
    pull = plan * slope * g.unsqueeze(1)
    return dict(loss=(plan * f).sum(1), grad_ratio=torch.cat([pull.sum(1), -pull.sum(0)]),
                grad_plan=f * g.unsqueeze(1))


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] in ("route", "balance"):
        rows, size = c["B"] * c["N"], _SIZE[c["dtype"]]
        live = rows * c["valid"]
        grad = c.get("grad", True)
        b = live * c["E"] * size + (c["B"] * c["E"] + c["B"]) * 4 + (rows if c["valid"] < 1.0 else 0)
        b += rows * c["k"] * (8 if c["kind"] == "route" else 4)  # weights and experts out, or experts in
        if grad:
            b += rows * c["E"] * size + c["B"] * 4 + (rows * c["k"] * 4 if c["kind"] == "route" else 0)
        return {"bytes": b, "flops": live * c["E"] * (12.0 if grad else 5.0)}
    if c["kind"] == "logp":
        rows, size = c["B"] * c["S"], _SIZE[c["dtype"]]
        live = rows * (0.55 if c["masked"] else 1.0)  # 0.2 of a sequence prompt, 0.25 padding on average
        b = live * c["V"] * size + rows * 8 + (rows if c["masked"] else 0) + c["B"] * 4
        if c["grad"]:
            b += rows * c["V"] * size
        return {"bytes": b, "flops": live * c["V"] * (8.0 if c["grad"] else 4.0)}
    pairs = c["P"] * c["Q"] if c["plan"] else c["P"]
    b = (c["P"] + c["Q"]) * 8 + c["P"] * 8 + (pairs * 8 if c["plan"] else 0)
    return {"bytes": b, "flops": pairs * 20.0}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "balance": _exact_balance, "logp": _exact_logp, "prefer": _exact_prefer}[
        case["kind"]](s)


def _exact_balance_loss(p, experts, mask, k):
    """Each batch element on its own: E times the product of the assigned and the mean share, summed."""
    losses, counts = [], []
    for b in range(p.shape[0]):
        rows = p[b] if mask is None else p[b][mask[b]]
        took = experts[b] if mask is None else experts[b][mask[b]]
        took = took.reshape(-1)
        hist = torch.bincount(took[took >= 0].long(), minlength=p.shape[2])
        n = max(rows.shape[0], 1)
        losses.append(p.shape[2] * (hist.double() / (k * n) * rows.sum(0) / n).sum())
        counts.append(hist)
    return torch.stack(losses), torch.stack(counts)


def _shares(x, scoring):
    if scoring == "softmax":
        q = torch.softmax(x, -1)
        return q, q
    q = torch.sigmoid(x) if scoring == "sigmoid" else x
    return q, q / q.sum(-1, keepdim=True)


def _exact_route(s):
    c = s["case"]
    x = s["scores"].detach().double().requires_grad_(c["grad"])
    key = s["scores"].detach().float()
    key = key if s["bias"] is None else key + s["bias"]  # the order is that of 32-bit keys
    experts = torch.argsort(-key, dim=-1, stable=True)[..., :c["k"]]
    q, p = _shares(x, c["scoring"])
    if c["normalize"] and c["scoring"] == "softmax":
        w = torch.softmax(x.gather(-1, experts), -1)
    else:
        w = q.gather(-1, experts)
        if c["normalize"]:
            w = w / w.sum(-1, keepdim=True)
    if s["mask"] is not None:
        gone = ~s["mask"].unsqueeze(-1)
        w = w.masked_fill(gone, 0.0)
        experts = experts.masked_fill(gone, -1)
    loss, counts = _exact_balance_loss(p, experts, s["mask"], c["k"])
    out = dict(weights=w.detach(), experts=experts.to(torch.int32), counts=counts.to(torch.int32),
               balance_loss=loss.detach())
    if c["grad"]:
        total = (w * s["grad_weights"].double()).sum() + (loss * s["grad_loss"].double()).sum()
        (out["grad_scores"],) = torch.autograd.grad(total, x)
    return out


def _exact_balance(s):
    c = s["case"]
    x = s["scores"].detach().double().requires_grad_()
    _, p = _shares(x, c["scoring"])
    loss, counts = _exact_balance_loss(p, s["experts"], s["mask"], c["k"])
    (g,) = torch.autograd.grad((loss * s["grad_loss"].double()).sum(), x)
    return dict(loss=loss.detach(), counts=counts.to(torch.int32), grad_scores=g)


def _exact_logp(s):
    c = s["case"]
    B, S, V = s["logits"].shape
    outs, grads = [], []
    for b in range(B):
        x = s["logits"][b].detach().double().requires_grad_(c["grad"])
        lp = torch.log_softmax(x / c["tau"], -1)[torch.arange(S, device=x.device), s["tokens"][b]]
        ref = s["ref"]
        if ref is not None and ref.dim() == 2:
            lp = lp - ref[b].double()
        m = torch.ones_like(lp, dtype=torch.bool) if s["mask"] is None else s["mask"][b]
        if c["reduction"] == "none":
            o = lp.masked_fill(~m, 0.0)
        else:
            o = lp[m].sum()
            if c["reduction"] == "mean":
                o = o / max(int(m.sum()), 1)
            if ref is not None and ref.dim() == 1:
                o = o - ref[b].double()
        outs.append(o.detach())
        if c["grad"]:
            (g,) = torch.autograd.grad((o * s["grad"][b].double()).sum(), x)
            grads.append(g)
        del x, lp, o
    out = dict(logp=torch.stack(outs))
    if c["grad"]:
        out["grad_logits"] = torch.stack(grads)
    return out


def _exact_prefer(s):
    c = s["case"]
    P = c["P"]
    r = s["ratio"].detach().double().requires_grad_()
    plan = s["plan"].detach().double().requires_grad_() if c["plan"] else None
    gap = r[:P, None] - r[None, P:] if c["plan"] else r[:P] - r[P:]
    d = c["beta"] * gap
    if c["loss_type"] == "sigmoid":
        f = -((1 - c["smoothing"]) * torch.nn.functional.logsigmoid(d)
              + c["smoothing"] * torch.nn.functional.logsigmoid(-d))
    elif c["loss_type"] == "hinge":
        f = torch.relu(1 - d)
    else:
        f = (gap - 1 / (2 * c["beta"])) ** 2
    loss = f if plan is None else (plan * f).sum(1)
    leaves = [r] if plan is None else [r, plan]
    grads = torch.autograd.grad((loss * s["grad"].double()).sum(), leaves)
    return dict(loss=loss.detach(), **dict(zip(("grad_ratio", "grad_plan"), grads)))
