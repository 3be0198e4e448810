"""Distillation from a teacher's top log-probabilities, and beam search: what is measured.

A case is a dict of plain values.  Its ``kind`` says which operator it runs:

* ``top``     — ``top_logp``: the k largest log-probabilities of each position and
  their tokens, from the logits (a teacher's targets; candidates shown to a user);
* ``distill`` — ``distill_loss``: divergence of a student's logits from a teacher's
  top log-probabilities, and the gradient of the logits;
* ``beam``    — ``beam_step``: the best continuations over beams and vocabulary;
* ``reorder`` — ``beam_reorder``: the states of the chosen beams, in place.

``own`` selects the framework's operators; without it ``run`` computes the
same from elementary operations in 32 bits (64 for long sums, for the few values
of a teacher's tokens, and for the totals that beams are compared by).
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "i64": torch.int64}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "i64": 8}
_MOST_LOGITS = 1 << 27  # elements of the largest logits that draw() makes (the largest listed case has 2^30)
_MOST_STATE = 1 << 28   # and of the largest states (the largest listed case has 2^29)


def _top(name, B, S, V, k, dtype, tau=1.0, masked=False):
    return dict(name=name, kind="top", B=B, S=S, V=V, k=k, dtype=dtype, tau=tau, masked=masked)


def _distill(name, B, S, V, k, dtype, tau=1.0, direction="forward", rest="bucket", reduction="mean", masked=True):
    return dict(name=name, kind="distill", B=B, S=S, V=V, k=k, dtype=dtype, tau=tau, direction=direction, rest=rest,
                reduction=reduction, masked=masked)


def _beam(name, B, W, V, n, dtype, tau=1.0, finished=0.0):
    return dict(name=name, kind="beam", B=B, W=W, V=V, n=n, dtype=dtype, tau=tau, finished=finished)


def _reorder(name, B, W, H, S, D, dtype, count, layout="heads", ragged=True):
    return dict(name=name, kind="reorder", B=B, W=W, H=H, S=S, D=D, dtype=dtype, count=count, layout=layout,
                ragged=ragged)


def listed():
    return [
        # Serving: the candidates of one decoding step of a few requests, shown beside the answer; latency.
        _top("top_decode", 8, 1, 32768, 20, "bf16"),
        # A teacher's targets for a batch of answers over a large vocabulary, short lists.
        _top("top_teacher", 4, 1024, 131072, 64, "bf16"),
        # Softened targets over an odd vocabulary, fp32, masked prompts, long lists.
        _top("top_odd", 3, 333, 50021, 128, "fp32", tau=2.0, masked=True),
        # A small student on a few short answers; latency.
        _distill("distill_small", 2, 37, 1000, 8, "fp32", masked=False),
        # Training on a batch of answers with masked prompts and padding.
        _distill("distill_train", 8, 1023, 32768, 64, "bf16"),
        # Mode-seeking distillation at a higher temperature over an odd vocabulary, fp32.
        _distill("distill_reverse", 6, 129, 50021, 100, "fp32", tau=2.0, direction="reverse", reduction="sum"),
        # Long answers over a large vocabulary, the teacher's list taken as the whole: the largest call.
        _distill("distill_long", 4, 2048, 131072, 128, "bf16", rest="none"),
        # One request with a few beams; latency.
        _beam("beam_decode", 1, 4, 32768, 4, "bf16"),
        # A batch of requests, two candidates for each beam, some hypotheses finished.
        _beam("beam_serve", 32, 8, 131072, 16, "bf16", finished=0.2),
        # Many beams over an odd vocabulary, fp32, sharpened.
        _beam("beam_odd", 5, 48, 50021, 96, "fp32", tau=0.7),
        # The tokens so far of a batch of hypotheses; latency.
        _reorder("reorder_tokens", 64, 8, 1, 513, 1, "i64", 1, layout="tokens", ragged=False),
        # Keys and values of eight layers, ragged lengths.
        _reorder("reorder_cache", 8, 4, 8, 1024, 128, "bf16", 16),
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(["top", "distill", "distill", "beam", "beam", "reorder"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    V = _log_uniform(rng, 1000, 160000)
    if rng.random() < 0.5:
        V = V // 64 * 64 + 64
    tau = rng.choice([1.0, 1.0, 0.6, 2.0])
    if kind in ("top", "distill"):
        B = rng.randint(1, 16)
        S = _log_uniform(rng, 1, max(1, min(4096, _MOST_LOGITS // (B * V))))
        k = _log_uniform(rng, 1, 256)
        masked = rng.random() < 0.6
        if kind == "top":
            return _top("", B, S, V, k, dtype, tau, masked)
        direction = rng.choice(["forward", "forward", "reverse"])
        rest = "bucket" if direction == "reverse" else rng.choice(["bucket", "bucket", "none"])
        return _distill("", B, S, V, k, dtype, tau, direction, rest, rng.choice(["sum", "mean", "none"]), masked)
    if kind == "beam":
        W = _log_uniform(rng, 1, 64)
        B = _log_uniform(rng, 1, max(1, min(64, _MOST_LOGITS // (W * V))))
        n = min(256, rng.choice([W, 2 * W, 2 * W + 1]))
        return _beam("", B, W, V, n, dtype, tau, rng.choice([0.0, 0.3]))
    W = _log_uniform(rng, 2, 32)
    B = _log_uniform(rng, 1, 32)
    if rng.random() < 0.3:
        return _reorder("", B, W, 1, _log_uniform(rng, 1, 4096), 1, "i64", 1, "tokens", rng.random() < 0.5)
    H, D = rng.choice([1, 2, 8]), rng.choice([64, 80, 128, 256])
    count = rng.choice([2, 8, 32])
    S = _log_uniform(rng, 1, max(1, min(4096, _MOST_STATE // (B * W * H * D * count))))
    return _reorder("", B, W, H, S, D, dtype, count, rng.choice(["heads", "positions"]), rng.random() < 0.7)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")  # the CPU: to look at the forms only
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    make = dict(device=dev, generator=gen)
    c = dict(case)
    return {"top": _prepare_top, "distill": _prepare_distill, "beam": _prepare_beam,
            "reorder": _prepare_reorder}[c["kind"]](c, dev, make)


def _logits(shape, c, make):
    """Logits of a trained model: a spread of 2, and a few tokens well above the others."""
    x = torch.randn(*shape, dtype=_DTYPES[c["dtype"]], **make).mul_(2.0)
    likely = torch.randint(0, shape[-1], (*shape[:-1], 4), **make)
    top = math.log(shape[-1]) + 6.0 * torch.rand(*shape[:-1], 4, **make)
    return x.scatter_(-1, likely, (c["tau"] * top).to(x.dtype))


def _answer_mask(B, S, dev, make):
    """Positions of answers: a prompt before, padding behind."""
    at = torch.arange(S, device=dev)
    prompt = (torch.rand(B, 1, **make) * 0.4 * S).long()
    end = ((0.5 + 0.5 * torch.rand(B, 1, **make)) * S).long() + 1
    return (at >= prompt) & (at < end)


def _prepare_top(c, dev, make):
    s = dict(case=c, logits=_logits((c["B"], c["S"], c["V"]), c, make), mask=None)
    if c["masked"]:
        s["mask"] = _answer_mask(c["B"], c["S"], dev, make)
    return s


def _prepare_distill(c, dev, make):
    B, S, V, k = c["B"], c["S"], c["V"], c["k"]
    s = dict(case=c, logits=_logits((B, S, V), c, make), mask=None)
    logp, tokens = [], []
    for b in range(B):
        # A teacher near this student: its logits to within about one.
        teacher = torch.randn(S, V, **make).add_(s["logits"][b]).div_(c["tau"])
        best = teacher.topk(k, dim=-1)
        logp.append(best.values - torch.logsumexp(teacher, -1, keepdim=True))
        tokens.append(best.indices)
    s["logp"], s["tokens"] = torch.stack(logp), torch.stack(tokens).to(torch.int32)
    if c["masked"]:
        s["mask"] = _answer_mask(B, S, dev, make)
    # the divergence enters the training loss with a weight of its own
    s["grad"] = torch.rand(B, S, **make) + 0.5 if c["reduction"] == "none" else torch.rand(B, **make) + 0.5
    s["logits"].requires_grad_()
    return s


def _prepare_beam(c, dev, make):
    B, W, V = c["B"], c["W"], c["V"]
    s = dict(case=c, logits=_logits((B, W, V), c, make), finished=None, eos=2)
    # Scores of hypotheses of some twenty tokens, the best first.
    s["scores"] = (-20.0 - 6.0 * torch.rand(B, W, **make)).sort(-1, descending=True).values
    if c["finished"]:
        s["finished"] = torch.rand(B, W, **make) < c["finished"]
    return s


def _prepare_reorder(c, dev, make):
    B, W, H, S, D = c["B"], c["W"], c["H"], c["S"], c["D"]
    shape = {"heads": (B, W, H, S, D), "positions": (B, W, S, H, D), "tokens": (B, W, S)}[c["layout"]]
    dim = {"heads": 3, "positions": 2, "tokens": 2}[c["layout"]]
    if c["dtype"] == "i64":
        states = [torch.randint(0, 32768, shape, **make) for _ in range(c["count"])]
    else:
        states = [torch.randn(*shape, dtype=_DTYPES[c["dtype"]], **make) for _ in range(c["count"])]
    # Parents of a step: the better beams have more children.
    beams = (W * torch.rand(B, W, **make).square()).int().clamp_(max=W - 1)
    s = dict(case=c, states=states, beams=beams, lengths=None, dim=dim)
    if c["ragged"]:
        s["lengths"] = ((0.5 + 0.5 * torch.rand(B, **make)) * S).int()
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"top": _own_top, "distill": _own_distill, "beam": _own_beam, "reorder": _own_reorder}[kind](state)
    return {"top": _plain_top, "distill": _plain_distill, "beam": _plain_beam, "reorder": _plain_reorder}[kind](state)


def _own_top(s):
    import dot_amd

    r = dot_amd.top_logp(s["logits"], s["case"]["k"], tau=s["case"]["tau"], mask=s["mask"])
    return dict(logp=r.logp, tokens=r.tokens)


def _own_distill(s):
    import dot_amd

    c = s["case"]
    loss = dot_amd.distill_loss(s["logits"], s["logp"], s["tokens"], mask=s["mask"], tau=c["tau"],
                                direction=c["direction"], rest=c["rest"], reduction=c["reduction"])
    (g,) = torch.autograd.grad([loss], [s["logits"]], [s["grad"]])
    return dict(loss=loss, grad_logits=g)


def _own_beam(s):
    import dot_amd

    c = s["case"]
    r = dot_amd.beam_step(s["logits"], s["scores"], k=c["n"], tau=c["tau"], finished=s["finished"], eos=s["eos"])
    return dict(scores=r.scores, beams=r.beams, tokens=r.tokens, finished=r.finished)


def _own_reorder(s):
    import dot_amd

    dot_amd.beam_reorder(s["states"], s["beams"], lengths=s["lengths"], dim=s["dim"])
    return s["states"]


# --- the plain form ---------------------------------------------------------
def _best(x, k):
    """Tokens of the k largest of each row, equal ones by the lowest index: a key of the value above the index."""
    bits = x.float().view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (order << 32) | (0xFFFFFFFF - torch.arange(x.shape[-1], device=x.device))
    return 0xFFFFFFFF - (key.topk(k, dim=-1).values & 0xFFFFFFFF)


def _plain_logp(x, tokens, tau):
    """Log-probabilities of some tokens of each row, in 64 bits."""
    z = x.float()
    if tau != 1.0:
        z = z / tau
    top = z.amax(-1, keepdim=True)
    total = torch.exp(z - top).sum(-1, keepdim=True, dtype=torch.float64)
    return (z.gather(-1, tokens) - top).double() - torch.log(total)


def _plain_top(s):
    c = s["case"]
    tokens = _best(s["logits"], c["k"])
    logp = _plain_logp(s["logits"], tokens, c["tau"]).float()
    if s["mask"] is not None:
        out = ~s["mask"].unsqueeze(-1)
        logp, tokens = logp.masked_fill(out, -math.inf), tokens.masked_fill(out, -1)
    return dict(logp=logp, tokens=tokens.int())


def _plain_distill(s):
    c = s["case"]
    at = s["tokens"].long()
    z = s["logits"].detach().float()
    if c["tau"] != 1.0:
        z = z / c["tau"]
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    # the teacher's few tokens in 64 bits, the others on their own: neither hides the digits of the other
    listed_e = torch.exp((z.gather(-1, at) - top).double())
    others = e.scatter(-1, at, 0.0).sum(-1, keepdim=True, dtype=torch.float64)
    log_total = torch.log(listed_e.sum(-1, keepdim=True) + others)
    log_q = (z.gather(-1, at) - top).double() - log_total
    log_qr = torch.log(others) - log_total
    q, qr = torch.exp(log_q), torch.exp(log_qr)
    t = s["logp"].double()
    p = torch.exp(t)
    mass = p.sum(-1, keepdim=True)
    if c["rest"] == "none":
        p, t = p / mass, t - torch.log(mass)
        value = (p * (t - log_q)).sum(-1)
        listed_grad, other_grad = q - p, qr
    else:
        pr = (1.0 - mass).clamp(min=0.0)
        if c["direction"] == "forward":
            value = (p * (t - log_q)).sum(-1) + (pr * (torch.log(pr.clamp(min=1e-300)) - log_qr)).squeeze(-1)
            listed_grad, other_grad = q - p, qr - pr
        else:
            log_pr = torch.log(pr.clamp(min=2.0**-24))
            value = (q * (log_q - t)).sum(-1) + (qr * (log_qr - log_pr)).squeeze(-1)
            listed_grad = q * (log_q - t - value.unsqueeze(-1))
            other_grad = qr * (log_qr - log_pr - value.unsqueeze(-1))
    keep = torch.ones_like(value) if s["mask"] is None else s["mask"].double()
    weight = keep
    loss = value * keep
    if c["reduction"] != "none":
        if c["reduction"] == "mean":
            weight = keep / keep.sum(1, keepdim=True).clamp(min=1.0)
        loss = (value * weight).sum(1)
    g = s["grad"] if c["reduction"] == "none" else s["grad"].unsqueeze(1)
    coef = (g * weight / c["tau"]).unsqueeze(-1)
    grad = e.mul_((coef * other_grad / others).float())
    grad.scatter_(-1, at, (coef * listed_grad).float())
    return dict(loss=loss.float(), grad_logits=grad.to(s["logits"].dtype))


def _plain_beam(s):
    c = s["case"]
    B, W, V, n = c["B"], c["W"], c["V"], c["n"]
    m = min(n, V)
    tokens = _best(s["logits"], m)
    total = s["scores"].double().unsqueeze(-1) + _plain_logp(s["logits"], tokens, c["tau"])
    done = s["finished"]
    if done is not None:
        # a finished hypothesis goes on as it is, once
        first = torch.arange(m, device=total.device) == 0
        same = torch.where(first, s["scores"].double().unsqueeze(-1), -math.inf)
        total = torch.where(done.unsqueeze(-1), same, total)
        tokens = torch.where(done.unsqueeze(-1), s["eos"], tokens)
    order = torch.sort(total.view(B, W * m), dim=-1, descending=True, stable=True)
    at, scores = order.indices[:, :n], order.values[:, :n]
    beams, tokens = at // m, tokens.view(B, W * m).gather(-1, at)
    finished = tokens == s["eos"]
    if done is not None:
        finished = finished | done.gather(-1, beams)
    none = scores == -math.inf  # fewer continuations than asked for
    beams, tokens = beams.masked_fill(none, -1), tokens.masked_fill(none, -1)
    return dict(scores=scores.float(), beams=beams.int(), tokens=tokens.int(), finished=finished & ~none)


def _plain_reorder(s):
    beams = s["beams"].long()
    batch = torch.arange(beams.shape[0], device=beams.device).unsqueeze(1)
    for t in s["states"]:
        new = t[batch, beams]
        if s["lengths"] is not None:
            shape = [1] * t.dim()
            shape[s["dim"]] = t.shape[s["dim"]]
            at = torch.arange(t.shape[s["dim"]], device=t.device).view(shape)
            new = torch.where(at < s["lengths"].view(-1, *[1] * (t.dim() - 1)), new, t)
        t.copy_(new)
    return s["states"]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] in ("top", "distill"):
        rows, size, k = c["B"] * c["S"], _SIZE[c["dtype"]], c["k"]
        # 0.2 of a sequence prompt, 0.25 padding on average; one position is never padding
        live = rows * (0.55 if c["masked"] and c["S"] > 1 else 1.0)
        b = live * c["V"] * size + (rows if c["masked"] else 0)
        if c["kind"] == "top":
            return {"bytes": b + rows * k * 8, "flops": live * c["V"] * 4.0}
        b += live * k * 8 + rows * c["V"] * size + (rows if c["reduction"] == "none" else c["B"]) * 8
        return {"bytes": b, "flops": live * c["V"] * 8.0}
    if c["kind"] == "beam":
        rows = c["B"] * c["W"] * (1.0 - c["finished"])
        return {"bytes": rows * c["V"] * _SIZE[c["dtype"]] + c["B"] * (c["W"] * 5 + c["n"] * 13),
                "flops": rows * c["V"] * 4.0}
    W = c["W"]
    share = [math.sqrt((j + 1) / W) - math.sqrt(j / W) for j in range(W)]  # of the children that beam j has
    written = sum(1.0 - p for p in share)
    read = sum(1.0 - (1.0 - p) ** (W - 1) for p in share)
    beam = c["H"] * c["S"] * c["D"] * _SIZE[c["dtype"]] * c["count"] * (0.75 if c["ragged"] else 1.0)
    return {"bytes": c["B"] * ((written + read) * beam + 4 * W), "flops": 0.0}


# ---------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"top": _exact_top, "distill": _exact_distill, "beam": _exact_beam,
            "reorder": _exact_reorder}[case["kind"]](s)


def _exact_top(s):
    c = s["case"]
    rows = []
    for b in range(c["B"]):
        p = torch.log_softmax(s["logits"][b].double() / c["tau"], -1).topk(c["k"], -1).values
        rows.append(p if s["mask"] is None else p.masked_fill(~s["mask"][b].unsqueeze(-1), -math.inf))
    return dict(logp=torch.stack(rows), tokens=None)


def _exact_distill(s):
    c = s["case"]
    losses, grads = [], []
    for b in range(c["B"]):
        x = s["logits"][b].detach().double().requires_grad_()
        logq = torch.log_softmax(x / c["tau"], -1)
        at, t = s["tokens"][b].long(), s["logp"][b].double()
        chosen = logq.gather(-1, at)
        inside = torch.zeros_like(logq, dtype=torch.bool).scatter_(-1, at, True)
        other = torch.logsumexp(logq.masked_fill(inside, -math.inf), -1)
        left = (1.0 - t.exp().sum(-1)).clamp(min=0.0)
        if c["rest"] == "none":
            target = torch.softmax(t, -1)
            d = (target * (torch.log_softmax(t, -1) - chosen)).sum(-1)
        elif c["direction"] == "forward":
            d = (t.exp() * (t - chosen)).sum(-1) + torch.special.xlogy(left, left) - left * other
        else:
            d = (chosen.exp() * (chosen - t)).sum(-1) + other.exp() * (other - left.clamp(min=2.0**-24).log())
        m = torch.ones_like(d, dtype=torch.bool) if s["mask"] is None else s["mask"][b]
        if c["reduction"] == "none":
            loss = d.masked_fill(~m, 0.0)
        else:
            loss = d[m].sum()
            if c["reduction"] == "mean":
                loss = loss / max(int(m.sum()), 1)
        losses.append(loss.detach())
        (g,) = torch.autograd.grad((loss * s["grad"][b].double()).sum(), x)
        grads.append(g)
        del x, logq, chosen, inside, other, d, loss
    return dict(loss=torch.stack(losses), grad_logits=torch.stack(grads))


def _exact_beam(s):
    c = s["case"]
    scores = []
    for b in range(c["B"]):
        total = s["scores"][b].double().unsqueeze(-1) + torch.log_softmax(s["logits"][b].double() / c["tau"], -1)
        if s["finished"] is not None:
            gone = s["finished"][b]
            total[gone] = -math.inf
            total[gone, s["eos"]] = s["scores"][b][gone].double()
        scores.append(total.view(-1).topk(c["n"]).values)
    return dict(scores=torch.stack(scores), beams=None, tokens=None, finished=None)


def _exact_reorder(s):
    out = []
    for t in s["states"]:
        new = t.clone()
        for b, parents in enumerate(s["beams"].tolist()):
            old, into = t[b], new[b]
            if s["lengths"] is not None:
                used = int(s["lengths"][b])
                old, into = old.narrow(s["dim"] - 1, 0, used), into.narrow(s["dim"] - 1, 0, used)
            for w, parent in enumerate(parents):
                into[w] = old[parent]
        out.append(new)
    return out
