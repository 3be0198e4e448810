"""Digits of the routing, sequence log-probability and preference operators on the
device, element by element against the float64 definition."""

import numpy as np
import pytest
import torch

import dot_amd
from oracle import training as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    """Relative, and absolute for results that are subnormal."""
    info = torch.finfo(dtype)
    return info.eps / 2, float(info.smallest_normal) * info.eps / 2


def taken_rows(rng, V, dtype):
    """(2, 12, V) logits: tokens from unlikely over even chances to nearly certain, and certain ones."""
    x = torch.as_tensor(rng.standard_normal((2, 12, V)).astype(np.float32))
    tokens = rng.integers(0, V, (2, 12))
    rest = float(np.log(max(V - 1, 1)) + 0.5)  # about the log of the others' sum
    for s in range(12):
        at = torch.as_tensor(tokens[:, s])[:, None]
        x[:, s].scatter_(1, at, rest + (-6.0, -1.0, -0.1, 0.0, 0.1, 1.0, 4.0, 8.0, 12.0, 16.0, 24.0, 0.0)[s])
    others = torch.ones(2, V, dtype=torch.bool).scatter_(1, torch.as_tensor(tokens[:, 11])[:, None], False)
    x[:, 11][others] = -float("inf")
    x[:, 3, :] = 1.5  # the same chance for all
    return x.to(dtype), tokens


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 8, 100, 4099, 40000, 131072])
def test_gradient_of_likely_tokens_keeps_its_digits(dtype, V):
    """dx of the taken token is c (1 - p): others / total, where the sum of the others is good to 1e-6 of itself (each
    term to 2^-22, partial sums to 2^-21) and 1 - p, the reciprocal, c and their product add 2^-24 each; a p of at most
    1/2 is good to 2e-6 of itself.  dx of the others is c p.  A logit d tau below the largest is off by d 2^-24 for the
    difference, as much for its product with log2(e) / tau, and 2^-22 for the exponential, c and their product; the sum
    by 2^-20: d 2^-23 + 2^-22 + 2^-20 of itself.  Each to half a step of its type."""
    print(f"[taken] {dtype} V={V}", flush=True)
    rng = np.random.default_rng(V)
    logits, tokens = taken_rows(rng, V, DTYPES[dtype])
    half, tiny = half_step(DTYPES[dtype])
    for tau, reduction in ((1.0, "none"), (0.7, "sum"), (1.3, "mean")):
        x = logits.to(DEV).requires_grad_()
        out = dot_amd.sequence_logp(x, torch.as_tensor(tokens).to(DEV), tau=tau, reduction=reduction)
        up = rng.uniform(0.5, 2.0, tuple(out.shape)).astype(np.float32)
        (g,) = torch.autograd.grad([out], [x], [torch.as_tensor(up).to(DEV)])
        z = logits.double() / tau
        at = torch.as_tensor(tokens)[..., None]
        own = z.gather(2, at)
        c = torch.as_tensor(up).double() / tau / (12 if reduction == "mean" else 1)
        c = c[..., None] if reduction == "none" else c[:, None, None]
        rest = torch.logsumexp(z.scatter(2, at, -float("inf")), -1, keepdim=True)
        total = torch.logaddexp(own, rest)
        want = -c * torch.exp(z - total)
        want.scatter_(2, at, c * torch.exp(rest - total))
        err = (g.detach().cpu().double() - want).abs()
        taken = torch.zeros_like(z, dtype=torch.bool).scatter_(2, at, True)
        d = z.amax(-1, keepdim=True) - torch.where(z == -float("inf"), z.amax(-1, keepdim=True), z)
        relative = half + torch.where(taken, 3e-6, d * 2.0**-23 + 2.0**-22 + 2.0**-20)
        over = err - relative * want.abs() - tiny - (2.0**-126 if dtype == "fp32" else 0)  # flushed exponentials
        assert (over <= 0).all(), [(m & (over > 0)).sum() for m in (taken, ~taken)]
        assert (g[:, 11] == 0).all()


def test_gradient_of_large_logits():
    """Rows beyond 2^31 elements, before and behind where the caches end, every entry to half a step: p is good to 5e-6
    of itself (see above; logits up to 19 below the largest)."""
    B, S, V = 5, 1024, 500000
    x = torch.empty(B, S, V, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(0))
    tokens = torch.randint(0, V, (B, S), device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    # the last 224 MB, 234 rows of 10^6 bytes, are read through the caches: rows from 4886 on
    rows = [(0, 0), (2, 700), (4, 789), (4, 790), (4, 1022), (4, 1023)]
    mask = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    large = [0, 1, 7, 8, V // 3, V // 2 - 1, V // 2, V - 9, V - 8, V - 1]
    for i, (b, s) in enumerate(rows):
        mask[b, s] = True
        x[b, s, large] = 10.0 + torch.arange(len(large), device=DEV).roll(i).bfloat16() / 4
        tokens[b, s] = (large + [int(tokens[b, s])])[2 * i]
    x.requires_grad_()
    out = dot_amd.sequence_logp(x, tokens, mask=mask, reduction="none")
    (g,) = torch.autograd.grad(out.sum(), x)
    half, tiny = half_step(torch.bfloat16)
    for b, s in rows:
        want = -torch.softmax(x[b, s].detach().double(), 0)
        t = int(tokens[b, s])
        want[t] += 1
        assert want[large].abs().min() > 1e-3
        assert ((g[b, s].double() - want).abs() <= (half + 5e-6) * want.abs() + tiny).all(), (b, s)
    g[mask] = 0
    assert not g.any()


@pytest.mark.parametrize("scoring,normalize", [("sigmoid", True), ("sigmoid", False), ("softmax", True),
                                               ("softmax", False)])
@pytest.mark.parametrize("E,k", [(16, 8), (61, 16), (256, 8), (1024, 12)])
def test_weights_far_below_one_keep_their_digits(scoring, normalize, E, k):
    """Sigmoid scores near -20 and softmax scores down to -40 under the largest.  A mass is off by 1.25 ulp of its
    exponential (1.5e-7) and, in a softmax, by d 2^-24 for the difference d to the largest score (of the row, or of the
    selected).  Normalised: the sum of up to 16 such by as much as its terms and 4 roundings (2.4e-7), the quotient by
    2^-24: 6e-7.  An unnormalised softmax weight is divided by the sum over the row, whose terms are off by
    (d + 2) 2^-23: with sum p d <= log E <= 7 below 1.1e-6, with its roundings 1.5e-6 in all."""
    rng = np.random.default_rng(E)
    s = (-20.0 - 2.0 * rng.random((1, 200, E))).astype(np.float32)
    if scoring == "softmax":
        s = np.where(rng.random((1, 200, E)) < 2.0 / E, -rng.random((1, 200, E)), -40.0 * rng.random((1, 200, E)))
        s = s.astype(np.float32)
    x = torch.as_tensor(s).to(DEV).requires_grad_()
    r = dot_amd.topk_routing(x, k, scoring=scoring, normalize=normalize)
    o = oracle.route(s, k, scoring, normalize)
    assert np.array_equal(r.experts.cpu().numpy(), o["experts"])
    err = np.abs(r.weights.detach().cpu().double().numpy() / o["weights"] - 1)
    if scoring == "softmax":
        picked = np.take_along_axis(s, o["experts"], -1).astype(np.float64)
        top = picked.max(-1, keepdims=True) if normalize else s.max(-1, keepdims=True)
        # normalised, the sum's terms have that error too, weighed by their share: sum p d <= log 16
        err -= (top - picked + (np.log(16) if normalize else 0)) * 2.0**-24
    assert err.max() < (1.5e-6 if (scoring, normalize) == ("softmax", False) else 6e-7), err.max()
    if scoring == "sigmoid" and not normalize:  # the slope t u^2 is t here, times the upstream gradient: 1.5e-7 + 2^-24
        dw = rng.uniform(0.5, 2.0, o["weights"].shape).astype(np.float32)
        (g,) = torch.autograd.grad([r.weights], [x], [torch.as_tensor(dw).to(DEV)])
        og = oracle.route_grad(s, k, o, scoring, normalize, grad_weights=dw)
        assert (np.abs(g.cpu().double().numpy() - og) <= 2.2e-7 * np.abs(og)).all()


@pytest.mark.parametrize("coupled", [False, True])
@pytest.mark.parametrize("beta", [0.1, 0.05, 0.3, 1 / 3, 1.7, 64.0])
def test_hinge_at_its_kink(coupled, beta):
    """Gaps within a few fp32 steps of 1 / beta, and at 1 / beta itself: the loss is 0 or not, and the slope -beta or 0,
    as in 64 bits.  The loss is rounded once (sums of 33 positive ones 2e-6), the slope to fp32."""
    steps = np.arange(-16, 17)
    low = (np.array([0.0, 1e-8, -1e-8, 1.0, 3.0, -7.0, 1e-3, 100.0])).astype(np.float32)
    if not coupled:
        high = (low[:, None].astype(np.float64) + 1 / beta).astype(np.float32)
        high = (high + np.spacing(high) * steps).astype(np.float32)
        ratio = np.concatenate([high.ravel(), np.repeat(low, len(steps))])
        plan = None
    else:
        mid = np.float32(1 / beta)
        high = (mid + np.spacing(mid) * steps).astype(np.float32)
        ratio = np.concatenate([high, low[:3]])
        plan = np.ones((len(high), 3), np.float32) / 4
    r = torch.as_tensor(ratio).to(DEV).requires_grad_()
    pl = None if plan is None else torch.as_tensor(plan).to(DEV).requires_grad_()
    loss = dot_amd.preference_loss(r, plan=pl, beta=beta, loss_type="hinge")
    o, gr, gp = oracle.preference(ratio, plan, beta, "hinge")
    if not coupled:
        assert (np.abs(loss.detach().cpu().double().numpy() - o) <= 2.0**-24 * o).all()
    grads = torch.autograd.grad(loss.sum(), [r] + ([] if pl is None else [pl]))
    got = grads[0].cpu().double().numpy()
    assert np.array_equal(got != 0, gr != 0) and (np.abs(got - gr) <= 2e-6 * np.abs(gr)).all()
    if coupled:
        assert (np.abs(loss.detach().cpu().double().numpy() - o) <= 2e-6 * o).all()
        assert (np.abs(grads[1].cpu().double().numpy() - gp) <= 2.0**-24 * gp).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V,S", [(300, 2048), (32768, 500), (131072, 100)])
@pytest.mark.parametrize("tau", [1.0, 0.7])
def test_positions_less_their_reference(dtype, V, S, tau):
    """The error of single positions, which a reference of the same value in fp64 lays bare.  A term p_v of the sum is
    off by d_v 2^-24 for the difference to the largest logit, as much for its product and 2^-23 for the exponential;
    it is rescaled for a new maximum, at 2^-23 a time, in its thread (say 5 times), its wave, its workgroup and for the
    join; a pack adds 3 roundings: (2 sum_v p_v d_v + 2 + 16 + 3) 2^-24 of the sum, that is, of its logarithm."""
    gen = torch.Generator(DEV).manual_seed(V)
    x = (2 * torch.randn(2, S, V, device=DEV, generator=gen)).to(DTYPES[dtype])
    tokens = torch.randint(0, V, (2, S), device=DEV, generator=gen)
    taken = float(np.log(V)) - 3 + 10 * torch.rand(2, S, 1, device=DEV, generator=gen)
    x.scatter_(2, tokens[..., None], taken.to(x.dtype))
    for b in range(2):
        z = x[b].double() / tau
        want = torch.log_softmax(z, -1)
        spread = (want.exp() * (z.amax(-1, keepdim=True) - z)).sum(-1)
        ref = want.gather(1, tokens[b][:, None])[:, 0]
        err = dot_amd.sequence_logp(x[b], tokens[b], ref_logp=ref, tau=tau, reduction="none").double().abs()
        assert (err <= (2 * spread + 21) * 2.0**-24).all(), err.max()
