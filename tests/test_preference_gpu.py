"""preference_loss on the device against the float64 definition, and the
operators together as a training step uses them.

Tolerances: beta d is rounded twice (2^-23 relative), f and its slope follow to
a few ulp each (series, reciprocal and exponential), so 2e-6 of a term; sums of
up to 4096 positive terms add 4e-6 at most.  1e-5 of the largest value covers
both.
"""

import numpy as np
import pytest
import torch

import dot_amd
from conftest import rel_err
from oracle import training as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TOL = 1e-5


def check(ratio, plan=None, beta=0.1, loss_type="sigmoid", smoothing=0.0, seed=0):
    rng = np.random.default_rng(seed)
    r = torch.as_tensor(ratio).to(DEV).requires_grad_()
    pl = None if plan is None else torch.as_tensor(plan).to(DEV).requires_grad_()
    loss = dot_amd.preference_loss(r, plan=pl, beta=beta, loss_type=loss_type, label_smoothing=smoothing)
    up = rng.uniform(0.5, 1.5, loss.shape).astype(np.float32)
    o, gr, gp = oracle.preference(ratio, plan, beta, loss_type, smoothing, up)
    assert loss.dtype == torch.float32
    assert rel_err(loss, o) < TOL
    grads = torch.autograd.grad([loss], [r] + ([] if pl is None else [pl]), [torch.as_tensor(up).to(DEV)])
    assert rel_err(grads[0], gr) < TOL
    if pl is not None:
        assert rel_err(grads[1], gp) < TOL
        (only,) = torch.autograd.grad([dot_amd.preference_loss(r, plan=pl.detach(), beta=beta, loss_type=loss_type,
                                                               label_smoothing=smoothing)], [r],
                                      [torch.as_tensor(up).to(DEV)])
        assert torch.equal(only, grads[0])
    return loss, grads


LOSSES = [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("square", 0.0)]


@pytest.mark.parametrize("P", [1, 2, 63, 255, 256, 1000, 4097])
@pytest.mark.parametrize("loss_type,smoothing", LOSSES)
def test_pairs(P, loss_type, smoothing):
    rng = np.random.default_rng(P)
    ratio = (6 * rng.standard_normal(2 * P)).astype(np.float32)
    check(ratio, beta=0.25, loss_type=loss_type, smoothing=smoothing)


@pytest.mark.parametrize("P,Q", [(1, 1), (1, 4096), (4096, 1), (3, 5), (33, 1024), (64, 64), (100, 1025), (777, 1301),
                                 (2500, 36), (5, 8200)])
@pytest.mark.parametrize("loss_type,smoothing", LOSSES)
def test_plans(P, Q, loss_type, smoothing):
    print(f"[prefer] P={P} Q={Q} {loss_type}", flush=True)
    rng = np.random.default_rng(P + Q)
    ratio = (6 * rng.standard_normal(P + Q)).astype(np.float32)
    plan = rng.random((P, Q)).astype(np.float32) ** 3
    plan[P // 2] = 0.0
    check(ratio, plan / P, beta=0.2, loss_type=loss_type, smoothing=smoothing)


def test_far_ratios():
    """Differences of any size: no overflow, the small side keeps its digits."""
    ratio = np.array([0, 50, 500, 5000, -5000, 1e30, 3.0, 0, 0, 0, 0, 0, 0, 3.0], np.float32)
    loss, (g,) = check(ratio, beta=1.0)
    got, want = loss.detach().cpu().double().numpy(), oracle.preference(ratio, beta=1.0)[0]
    near = want > 1e-35
    assert (np.abs(got - want)[near] <= 1e-5 * want[near]).all()
    assert torch.isfinite(loss).all() and torch.isfinite(g).all()
    inf = torch.tensor([float("inf"), -float("inf"), 0.0, 0.0], device=DEV, requires_grad=True)
    loss = dot_amd.preference_loss(inf)
    (g,) = torch.autograd.grad(loss.sum(), inf)
    assert loss.tolist() == [0.0, float("inf")] and torch.isfinite(g).all()
    for loss_type in ("sigmoid", "hinge", "square"):
        nan = torch.tensor([float("nan"), 1.0, 0.0, 0.0], device=DEV)
        assert torch.isnan(dot_amd.preference_loss(nan, loss_type=loss_type)).tolist() == [True, False]


@pytest.mark.parametrize("loss_type,smoothing", LOSSES)
@pytest.mark.parametrize("P,Q", [(7, 12), (40, 1030)])
def test_pairs_left_out(P, Q, loss_type, smoothing):
    """Answers without a share of the plan may hold anything."""
    rng = np.random.default_rng(P)
    ratio = rng.standard_normal(P + Q).astype(np.float32)
    plan = rng.random((P, Q)).astype(np.float32) / P
    clean = ratio.copy()
    for at, value in ((1, np.nan), (3, np.inf), (5, -np.inf)):
        ratio[at] = ratio[P + at] = value
        clean[at] = clean[P + at] = 0.0
        plan[at] = 0.0
        plan[:, at] = 0.0
    with np.errstate(invalid="ignore"):
        loss, (g, gp) = check(ratio, plan, beta=0.3, loss_type=loss_type, smoothing=smoothing)
    want, (gc, _) = check(clean, plan, beta=0.3, loss_type=loss_type, smoothing=smoothing)
    assert torch.equal(loss, want) and torch.equal(g, gc)
    assert torch.isfinite(gp).all() and (loss[[1, 3, 5]] == 0).all()
    # weights of any size beside the ones left out
    check(ratio, np.where(plan == 0, 0, 1e30 * plan).astype(np.float32), beta=0.3, loss_type=loss_type,
          smoothing=smoothing)


def test_types_and_layouts():
    rng = np.random.default_rng(1)
    ratio = torch.as_tensor(rng.standard_normal(20).astype(np.float32)).to(DEV)
    plan = torch.as_tensor(rng.random((10, 10)).astype(np.float32)).to(DEV)
    base = dot_amd.preference_loss(ratio, plan=plan)
    assert torch.equal(dot_amd.preference_loss(ratio.repeat_interleave(2)[::2], plan=plan), base)
    assert torch.equal(dot_amd.preference_loss(ratio, plan=plan.t().contiguous().t()), base)
    half = plan.to(torch.bfloat16).requires_grad_()
    r64 = ratio.double().requires_grad_()
    loss = dot_amd.preference_loss(r64, plan=half)
    gr, gp = torch.autograd.grad(loss.sum(), [r64, half])
    assert loss.dtype == torch.float32 and gr.dtype == torch.float64 and gp.dtype == torch.bfloat16
    offset = torch.zeros(101, device=DEV)[1:].copy_(plan.reshape(-1)).view(10, 10)  # rows not 16-byte aligned
    assert rel_err(dot_amd.preference_loss(ratio, plan=offset), base) < TOL


def test_empty():
    z = torch.zeros(0, device=DEV, requires_grad=True)
    assert dot_amd.preference_loss(z).shape == (0,)
    for P, Q in ((3, 0), (0, 3)):
        r = torch.ones(3, device=DEV, requires_grad=True)
        plan = torch.zeros(P, Q, device=DEV, requires_grad=True)
        loss = dot_amd.preference_loss(r, plan=plan)
        g, gp = torch.autograd.grad(loss.sum(), [r, plan])
        assert (loss == 0).all() and (g == 0).all() and gp.shape == (P, Q)


def test_same_bits_twice():
    r = torch.randn(6000, device=DEV, generator=torch.Generator(DEV).manual_seed(0)).requires_grad_()
    plan = torch.rand(2500, 3500, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).requires_grad_()
    runs = []
    for _ in range(2):
        loss = dot_amd.preference_loss(r, plan=plan)
        runs.append((loss, *torch.autograd.grad(loss.sum(), [r, plan])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
def test_balanced_routing_over_a_transport_plan():
    """Router logits -> balanced plan -> experts and weights -> balance loss of the logits, one gradient through all."""
    gen = torch.Generator().manual_seed(0)
    B, N, E, k = 2, 96, 16, 2
    logits = torch.randn(B, N, E, generator=gen)
    logits[..., :3] += 2.0  # experts that every token likes
    x = logits.to(DEV).requires_grad_()
    plan = dot_amd.sinkhorn_from_scores(x, tau=0.5, n_iters=200)
    r = dot_amd.topk_routing(plan, k, scoring="plan", normalize=True)
    q = dot_amd.balance_loss(x, r.experts)
    dw = torch.randn(r.weights.shape, generator=gen)
    total = (r.weights * dw.to(DEV)).sum() + 0.01 * q.loss.sum()
    (g,) = torch.autograd.grad(total, x)

    y = logits.to(DEV).requires_grad_()
    plan2 = dot_amd.sinkhorn_from_scores(y, tau=0.5, n_iters=200)
    top = torch.topk(plan2, k, dim=-1)
    w = top.values / top.values.sum(-1, keepdim=True)
    counts = torch.stack([torch.bincount(t.reshape(-1), minlength=E) for t in top.indices])
    loss = E * (counts / (k * N) * torch.softmax(y, -1).mean(1)).sum(-1)
    (want,) = torch.autograd.grad((w * dw.to(DEV)).sum() + 0.01 * loss.sum(), y)
    assert torch.equal(r.counts.long(), counts) and torch.equal(q.counts, r.counts)
    assert rel_err(r.weights, w) < TOL and rel_err(q.loss, loss) < TOL and rel_err(g, want) < 1e-4
    # the plan spreads what the logits alone would send to three experts
    assert int(r.counts.max()) < int(dot_amd.topk_routing(x, k).counts.max())


def test_preference_over_a_transport_plan():
    """Logits of two sets of answers -> log ratios -> plan between them -> loss; the gradient reaches the logits."""
    gen = torch.Generator().manual_seed(1)
    P, Q, S, V = 6, 10, 24, 700
    logits = torch.randn(P + Q, S, V, generator=gen)
    tokens = torch.randint(0, V, (P + Q, S), generator=gen)
    mask = torch.rand(P + Q, S, generator=gen) < 0.8
    ref = torch.log_softmax(logits, -1).gather(2, tokens[..., None])[..., 0] + 0.1 * torch.randn(P + Q, S, generator=gen)
    x = logits.to(DEV).requires_grad_()
    ratio = dot_amd.sequence_logp(x, tokens.to(DEV), ref_logp=ref.to(DEV), mask=mask.to(DEV))
    cost = torch.nn.functional.softplus(-0.5 * (ratio[:P, None] - ratio[None, P:]))
    plan = dot_amd.sinkhorn(cost, reg=0.2, n_iters=300).transport_plan
    loss = dot_amd.preference_loss(ratio, plan=plan, beta=0.5)
    (g,) = torch.autograd.grad(loss.sum(), x)

    y = logits.to(DEV).requires_grad_()
    lp = torch.log_softmax(y, -1).gather(2, tokens.to(DEV)[..., None])[..., 0] - ref.to(DEV)
    rho = (lp * mask.to(DEV)).sum(1)
    cost = torch.nn.functional.softplus(-0.5 * (rho[:P, None] - rho[None, P:]))
    plan2 = dot_amd.sinkhorn(cost, reg=0.2, n_iters=300).transport_plan
    want = (plan2 * cost).sum(1)
    (gw,) = torch.autograd.grad(want.sum(), y)
    # log ratios of order 1 from positions that are off by 4e-6 each; the plan's gradient is that of 300 sweeps
    assert rel_err(loss, want) < 1e-4 and rel_err(g, gw) < 1e-3


def test_training_step_in_a_graph():
    """Routing, log ratios and the loss of a step captured together and replayed."""
    gen = torch.Generator().manual_seed(2)
    data = [(torch.randn(2, 64, 32, generator=gen).to(DEV), torch.randn(4, 20, 500, generator=gen).to(DEV))
            for _ in range(3)]
    tokens = torch.randint(0, 500, (4, 20), generator=gen).to(DEV)

    def step(scores, logits):
        s, x = scores.detach().requires_grad_(), logits.detach().requires_grad_()
        r = dot_amd.topk_routing(s, 2)
        loss = dot_amd.preference_loss(dot_amd.sequence_logp(x, tokens))
        gs, gx = torch.autograd.grad(loss.mean() + 0.01 * r.balance_loss.mean() + r.weights[..., 0].mean(), [s, x])
        return r.experts, r.balance_loss.detach(), loss.detach(), gs, gx

    eager = [step(*d) for d in data]
    hs, hx = data[0][0].clone(), data[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(hs, hx)
        step(hs, hx)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(hs, hx)
    for i in (1, 2, 0, 1):
        hs.copy_(data[i][0])
        hx.copy_(data[i][1])
        graph.replay()
        torch.cuda.synchronize()
        between = step(*data[(i + 2) % 3])
        assert all(torch.equal(a, b) for a, b in zip(outs, eager[i]))
        assert all(torch.equal(a, b) for a, b in zip(between, eager[(i + 2) % 3]))


def test_two_streams_at_once_and_no_gradients():
    """Calls of two streams in flight together, and calls that record nothing, give the same bits."""
    gen = torch.Generator().manual_seed(3)
    data = [(torch.randn(2, 5000, 48, generator=gen).to(DEV), torch.randn(3, 40, 4000, generator=gen).bfloat16().to(DEV))
            for _ in range(2)]
    tokens = torch.randint(0, 4000, (3, 40), generator=gen).to(DEV)
    plan = torch.rand(40, 80, generator=gen).to(DEV)

    def step(scores, logits):
        r = dot_amd.topk_routing(scores, 4, normalize=True)
        per = dot_amd.sequence_logp(logits, tokens, reduction="none")
        loss = dot_amd.preference_loss(per.reshape(-1), plan=plan)
        return [x.detach() for x in (r.weights, r.experts, r.counts, r.balance_loss, per, loss)]

    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(*data[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, g in zip(want, got) for a, b in zip(w, g))
    leaves = [x.clone().requires_grad_() for x in data[0]]
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(want[0], step(*leaves)))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(want[0], step(*leaves)))
    # a second backward through one graph, and an unused output
    r = dot_amd.topk_routing(leaves[0], 4)
    (a,) = torch.autograd.grad(r.balance_loss.sum(), leaves[0], retain_graph=True)
    (b,) = torch.autograd.grad(r.balance_loss.sum(), leaves[0])
    assert torch.equal(a, b) and not r.experts.requires_grad and not r.counts.requires_grad
