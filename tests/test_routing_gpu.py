"""topk_routing and balance_loss on the device against the float64 definition.

Tolerances: masses and shares go through one hardware exponential whose
argument is rounded once, so their relative error is at most (|d| + 8) 2^-24
for scores d below the row's largest (2e-6 for the d <= 30 of these inputs);
sums of up to 4096 of them and the two products of the gradient stay below
1e-5 of the largest value.  A gradient in 16 bits adds half a step of its type.
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
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def grad_tol(dtype):
    return TOL + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def make_scores(rng, B, N, E, scoring, dtype):
    s = rng.standard_normal((B, N, E)) + 0.5 * rng.standard_normal(E)
    if scoring == "plan":
        e = np.exp(2 * s)
        s = e / e.sum(-1, keepdims=True) / max(N, 1)
    return torch.as_tensor(s.astype(np.float32)).to(dtype)


def check(scores, k, scoring="softmax", normalize=False, bias=None, mask=None, use=("weights", "loss"), seed=0):
    """One call and its gradient on the device against the oracle."""
    dtype = scores.dtype
    rng = np.random.default_rng(seed)
    x = scores.to(DEV).detach().requires_grad_()
    r = dot_amd.topk_routing(x, k, scoring=scoring, normalize=normalize,
                             bias=None if bias is None else torch.as_tensor(bias).to(DEV),
                             mask=None if mask is None else torch.as_tensor(mask).to(DEV))
    s = scores.float().numpy()
    o = oracle.route(s, k, scoring, normalize, bias, mask)
    assert r.weights.dtype == torch.float32 and r.experts.dtype == torch.int32 and r.counts.dtype == torch.int32
    assert np.array_equal(r.experts.cpu().numpy(), o["experts"])
    assert np.array_equal(r.counts.cpu().numpy(), o["counts"])
    assert rel_err(r.weights, o["weights"]) < TOL
    assert rel_err(r.balance_loss, o["loss"]) < TOL
    dw = rng.standard_normal(o["weights"].shape).astype(np.float32) if "weights" in use else None
    dl = rng.uniform(0.5, 1.5, o["loss"].shape).astype(np.float32) if "loss" in use else None
    outs, ups = [], []
    if dw is not None:
        outs.append(r.weights)
        ups.append(torch.as_tensor(dw).to(DEV))
    if dl is not None:
        outs.append(r.balance_loss)
        ups.append(torch.as_tensor(dl).to(DEV))
    (g,) = torch.autograd.grad(outs, [x], ups)
    assert g.dtype == dtype
    og = oracle.route_grad(s, k, o, scoring, normalize, mask, dw, dl)
    assert rel_err(g.float(), og) < grad_tol(dtype)
    return r, g


@pytest.mark.parametrize("E,k", [(1, 1), (3, 2), (8, 2), (8, 8), (16, 4), (24, 3), (61, 3), (64, 6), (128, 64), (200, 5),
                                 (256, 8), (500, 7), (512, 16), (1000, 2), (1024, 4), (2048, 3), (4095, 2), (4096, 64)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "plan"])
def test_experts(E, k, scoring):
    print(f"[routing] E={E} k={k} {scoring}", flush=True)
    rng = np.random.default_rng(E + k)
    N = 37 if E <= 512 else 9
    scores = make_scores(rng, 2, N, E, scoring, torch.float32)
    check(scores, k, scoring, normalize=False)
    check(scores, k, scoring, normalize=True)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("B,N,E,k", [(1, 1, 64, 4), (5, 3, 64, 4), (1, 1000, 16, 2), (2, 777, 61, 3), (3, 130, 256, 8)])
@pytest.mark.parametrize("scoring,normalize", [("softmax", False), ("softmax", True), ("sigmoid", False),
                                               ("sigmoid", True)])
def test_types_and_lengths(dtype, B, N, E, k, scoring, normalize):
    print(f"[routing] {dtype} B={B} N={N} E={E} k={k} {scoring} {normalize}", flush=True)
    rng = np.random.default_rng(N)
    scores = make_scores(rng, B, N, E, scoring, DTYPES[dtype])
    bias = (0.3 * rng.standard_normal(E)).astype(np.float32)
    mask = rng.random((B, N)) < 0.6
    mask[0] = B == 1  # a batch element without tokens
    check(scores, k, scoring, normalize, bias=bias, mask=mask)


@pytest.mark.parametrize("use", [("weights",), ("loss",)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "plan"])
@pytest.mark.parametrize("normalize", [False, True])
def test_one_output_in_the_loss(use, scoring, normalize):
    rng = np.random.default_rng(3)
    check(make_scores(rng, 2, 50, 40, scoring, torch.float32), 3, scoring, normalize, use=use)


def test_ties_go_to_the_lowest_index():
    rng = np.random.default_rng(4)
    for E in (8, 60, 256, 1024):
        scores = torch.as_tensor(rng.integers(-2, 3, (2, 33, E)).astype(np.float32))
        scores[0, 0] = 0.0
        scores[0, 1, ::2] = -0.0  # equal to 0
        scores[0, 1, 1::2] = 0.0
        for dtype in DTYPES.values():
            check(scores.to(dtype), min(E, 12))


def test_near_ties():
    """Keys that differ in their last bits, among many equal ones, with and without a bias."""
    rng = np.random.default_rng(11)
    for E in (8, 61, 256, 1024, 4096):
        k = min(E, 16)
        near = torch.as_tensor((1 + rng.integers(0, 40, (2, 9, E)) * 2.0**-23).astype(np.float32))
        near[0, 0] *= -1
        near[1, 3] = torch.as_tensor(rng.standard_normal(E).astype(np.float32))
        check(near, k, normalize=True)
        check(near, k, "sigmoid", bias=(rng.integers(-1, 2, E) * 2.0**-24).astype(np.float32))
        for dtype in (torch.float16, torch.bfloat16):  # every 16-bit value next to its neighbours
            eps = torch.finfo(dtype).eps
            half = torch.as_tensor((1 + rng.integers(-3, 4, (2, 9, E)) * eps / 2).astype(np.float32)).to(dtype)
            half[0, 1] = half[0, 1] * torch.finfo(dtype).smallest_normal * eps * 3  # denormals
            check(half, k)
            check(half, k, bias=(rng.standard_normal(E) * 1e-6).astype(np.float32))


def test_many_batch_elements():
    """More batch elements than one grid dimension holds."""
    B = 70001
    x = torch.randn(B, 2, 8, device=DEV, generator=torch.Generator(DEV).manual_seed(0)).requires_grad_()
    r = dot_amd.topk_routing(x, 2)
    (g,) = torch.autograd.grad(r.balance_loss.sum(), x)
    d = x.detach().double()
    p = torch.softmax(d, -1)
    counts = torch.zeros(B, 8, dtype=torch.int32, device=DEV)
    counts.scatter_add_(1, r.experts.flatten(1).long(), torch.ones(B, 4, dtype=torch.int32, device=DEV))
    assert torch.equal(r.counts, counts)
    h = 8 * counts.double() / (2 * 2)  # E counts / (k n)
    assert rel_err(r.balance_loss, (h * p.mean(1)).sum(1)) < TOL
    h = h[:, None] / 2
    assert rel_err(g, p * (h - (p * h).sum(-1, keepdim=True))) < TOL


def test_unavailable_experts():
    """-inf scores are never taken; a token without experts has none; a row of the lowest value is a row like others."""
    rng = np.random.default_rng(5)
    for dtype in DTYPES.values():
        scores = make_scores(rng, 2, 12, 24, "softmax", torch.float32).to(dtype)
        scores[0, 0] = -float("inf")
        scores[0, 1] = -float("inf")
        scores[0, 1, 7] = 0.5
        scores[0, 2, :20] = -float("inf")
        scores[0, 3] = torch.finfo(dtype).min
        scores[0, 4, 3:] = torch.finfo(dtype).min
        for normalize in (False, True):
            r, g = check(scores, 5, "softmax", normalize)
            assert (r.experts[0, 0] == -1).all() and (r.weights[0, 0] == 0).all() and (g[0, 0] == 0).all()
            assert r.experts[0, 1].tolist() == [7, -1, -1, -1, -1]
            check(scores, 5, "sigmoid", normalize)
        # a bias of -inf closes an expert for the selection alone
        bias = np.zeros(24, np.float32)
        bias[:22] = -np.inf
        r, _ = check(scores, 5, "softmax", False, bias=bias)
        assert r.experts.max() <= 23 and (r.experts[1, :, 2:] == -1).all()
    plan = make_scores(rng, 1, 9, 16, "plan", torch.float32)
    plan[0, 2] = 0.0  # a row that the plan gives nothing
    plan[0, 3, 2:] = 0.0
    for normalize in (False, True):
        r, g = check(plan, 4, "plan", normalize)
        assert (r.experts[0, 2] == -1).all() and (g[0, 2] == 0).all()
        shut = np.zeros(16, np.float32)
        shut[:14] = -np.inf
        r, _ = check(plan, 4, "plan", normalize, bias=shut)
        assert not ((r.experts >= 0) & (r.experts < 14)).any()
    plan[0, 4] = 1e-42  # masses that no fp32 reciprocal holds
    r = dot_amd.topk_routing(plan.to(DEV), 4, scoring="plan", normalize=True)
    assert torch.isfinite(r.weights).all() and torch.isfinite(r.balance_loss).all()


def test_a_single_expert_has_no_weight_gradient():
    """k = 1, normalised: the weight is exactly 1, so that only the balance loss moves the scores."""
    rng = np.random.default_rng(12)
    for scoring in ("softmax", "sigmoid", "plan"):
        scores = make_scores(rng, 2, 400, 24, scoring, torch.float32)
        r, _ = check(scores, 1, scoring, True)
        assert (r.weights == 1).all()


def test_masked_tokens_are_not_read():
    rng = np.random.default_rng(6)
    for scoring in ("softmax", "sigmoid", "plan"):
        for E in (16, 61, 256):
            scores = make_scores(rng, 2, 40, E, scoring, torch.float32)
            mask = rng.random((2, 40)) < 0.5
            mask[1] = False
            clean = dot_amd.topk_routing(scores.to(DEV), 3, scoring=scoring, mask=torch.as_tensor(mask).to(DEV))
            dirty = scores.clone()
            dirty[~torch.as_tensor(mask)] = float("nan")
            dirty[0, np.flatnonzero(~mask[0])[:3]] = float("inf")
            x = dirty.to(DEV).requires_grad_()
            r = dot_amd.topk_routing(x, 3, scoring=scoring, mask=torch.as_tensor(mask).to(DEV))
            (g,) = torch.autograd.grad([r.weights.sum() + r.balance_loss.sum()], [x])
            for a, c in ((r.weights, clean.weights), (r.experts, clean.experts), (r.counts, clean.counts),
                         (r.balance_loss, clean.balance_loss)):
                assert torch.equal(a, c)
            assert torch.isfinite(g).all() and (g[~torch.as_tensor(mask).to(DEV)] == 0).all()
            assert r.balance_loss[1] == 0 and (r.counts[1] == 0).all()


def test_nan_shows():
    """NaN is never selected and reaches the token's softmax weights and the loss, and nothing else."""
    rng = np.random.default_rng(7)
    scores = make_scores(rng, 2, 10, 32, "softmax", torch.float32)
    scores[0, 4, 9] = float("nan")
    for normalize in (False, True):
        r = dot_amd.topk_routing(scores.to(DEV), 4, normalize=normalize)
        assert torch.isnan(r.weights[0, 4]).all() and not (r.experts[0, 4] == 9).any() and (r.experts >= 0).all()
        assert torch.isnan(r.balance_loss).tolist() == [True, False]
        rest = torch.ones(2, 10, dtype=torch.bool)
        rest[0, 4] = False
        assert torch.isfinite(r.weights.cpu()[rest]).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype):
    """Strides other than the contiguous ones, odd offsets, broadcast rows, no batch dimension."""
    rng = np.random.default_rng(8)
    base = make_scores(rng, 6, 90, 80, "softmax", DTYPES[dtype])
    views = {
        "rows": lambda t: t[::2, 1::3, :64],
        "offset": lambda t: t[:, :, 1:65],
        "transposed batch": lambda t: t.transpose(0, 1)[:5],
        "columns": lambda t: t[:, :, ::2],
        "last first": lambda t: t[:, :40, :].permute(0, 2, 1)[:, :, :40],
        "broadcast": lambda t: t[:1, :, :64].expand(4, 90, 64),
    }
    for name, view in views.items():
        print(f"[routing] {dtype} {name}", flush=True)
        x = view(base.to(DEV)).detach().requires_grad_()
        assert name == "contiguous" or not x.is_contiguous()
        r = dot_amd.topk_routing(x, 3, normalize=True)
        (g,) = torch.autograd.grad([r.weights, r.balance_loss], [x],
                                   [torch.ones_like(r.weights) * torch.arange(3, device=DEV), r.balance_loss.detach()])
        y = view(base).contiguous().to(DEV).requires_grad_()
        rc = dot_amd.topk_routing(y, 3, normalize=True)
        (gc,) = torch.autograd.grad([rc.weights, rc.balance_loss], [y],
                                    [torch.ones_like(r.weights) * torch.arange(3, device=DEV), rc.balance_loss.detach()])
        assert torch.equal(r.experts, rc.experts) and torch.equal(r.counts, rc.counts)
        assert rel_err(r.weights, rc.weights) < TOL and rel_err(r.balance_loss, rc.balance_loss) < TOL
        assert rel_err(g.float(), gc.float()) < 2 * grad_tol(DTYPES[dtype])
    flat = base[0].to(DEV).requires_grad_()
    r2 = dot_amd.topk_routing(flat, 2)
    r3 = dot_amd.topk_routing(base[:1].to(DEV), 2)
    assert r2.weights.shape == (90, 2) and r2.counts.shape == (80,) and r2.balance_loss.shape == ()
    assert torch.equal(r2.weights, r3.weights[0]) and torch.equal(r2.balance_loss, r3.balance_loss[0])
    r2.balance_loss.backward()
    assert flat.grad.shape == flat.shape


def test_empty():
    for B, N in ((0, 5), (3, 0), (0, 0)):
        x = torch.zeros(B, N, 16, device=DEV, requires_grad=True)
        r = dot_amd.topk_routing(x, 2)
        assert r.weights.shape == (B, N, 2) and (r.counts == 0).all() and (r.balance_loss == 0).all()
        (g,) = torch.autograd.grad(r.weights.sum() + r.balance_loss.sum(), x)
        assert g.shape == x.shape
        q = dot_amd.balance_loss(x, torch.zeros(B, N, 2, dtype=torch.int64, device=DEV))
        assert (q.loss == 0).all() and q.counts.shape == (B, 16)


@pytest.mark.parametrize("int_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "plan"])
@pytest.mark.parametrize("B,N,E,k", [(2, 300, 8, 2), (1, 999, 61, 6), (3, 64, 300, 9)])
def test_balance_loss(int_type, scoring, B, N, E, k):
    rng = np.random.default_rng(E)
    for dtype in (torch.float32, torch.bfloat16):
        scores = make_scores(rng, B, N, E, scoring, dtype)
        given = rng.integers(-1, E, (B, N, k))
        given[0, 0] = E          # outside: not counted
        given[0, 1] = E - 1      # the same expert k times
        if int_type == torch.int64:
            given[0, 2] = 2**32  # outside in 64 bits, 0 in 32
        mask = rng.random((B, N)) < 0.7
        x = scores.to(DEV).requires_grad_()
        r = dot_amd.balance_loss(x, torch.as_tensor(given).to(int_type).to(DEV), scoring=scoring,
                                 mask=torch.as_tensor(mask).to(DEV))
        s = scores.float().numpy()
        o = oracle.route(s, k, scoring, mask=mask, given=given)
        assert np.array_equal(r.counts.cpu().numpy(), o["counts"])
        assert rel_err(r.loss, o["loss"]) < TOL
        dl = rng.uniform(0.5, 1.5, B)
        (g,) = torch.autograd.grad([r.loss], [x], [torch.as_tensor(dl).float().to(DEV)])
        og = oracle.route_grad(s, k, o, scoring, mask=mask, grad_loss=dl.astype(np.float32))
        assert rel_err(g.float(), og) < grad_tol(dtype)


def test_long_batch():
    """More tokens than one pass of the grid takes, all scorings of one assignment, and the same bits twice."""
    rng = np.random.default_rng(9)
    scores = torch.randn(2, 40011, 64, generator=torch.Generator().manual_seed(9))
    x = scores.to(DEV).requires_grad_()
    r = dot_amd.topk_routing(x, 4, normalize=True)
    (g,) = torch.autograd.grad(r.balance_loss.sum(), x)
    again = dot_amd.topk_routing(x, 4, normalize=True)
    (g2,) = torch.autograd.grad(again.balance_loss.sum(), x)
    for a, b in ((r.weights, again.weights), (r.experts, again.experts), (r.balance_loss, again.balance_loss), (g, g2)):
        assert torch.equal(a, b)
    d = scores.double()
    p = torch.softmax(d, -1)
    top = torch.argsort(-d, dim=-1, stable=True)[..., :4]  # torch.topk leaves the order of equal scores open
    counts = torch.stack([torch.bincount(t.reshape(-1), minlength=64) for t in top])
    assert torch.equal(r.counts.cpu().long(), counts)
    loss = 64 * (counts.double() / (4 * 40011) * p.mean(1)).sum(1)
    assert rel_err(r.balance_loss, loss) < TOL
    h = 64 * counts.double() / (4 * 40011.0**2)
    og = p * (h[:, None] - (p * h[:, None]).sum(-1, keepdim=True))
    assert rel_err(g, og) < TOL


def test_other_stream_and_graph():
    """On a side stream, and captured and replayed with the program's own calls between."""
    rng = np.random.default_rng(10)
    inputs = [make_scores(rng, 3, 500, 64, "softmax", torch.bfloat16).to(DEV) for _ in range(3)]

    def step(s):
        x = s.detach().requires_grad_()
        r = dot_amd.topk_routing(x, 4, normalize=True)
        (g,) = torch.autograd.grad(r.weights[..., 0].sum() + r.balance_loss.sum(), x)
        return r.weights.detach(), r.experts, r.counts, r.balance_loss.detach(), g

    eager = [step(s) for s in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    held = inputs[0].clone()
    with torch.cuda.stream(side):
        other = step(held)
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, eager[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held)
    for i in (1, 2, 0, 2):
        held.copy_(inputs[i])
        graph.replay()
        torch.cuda.synchronize()
        between = step(inputs[(i + 1) % 3])
        assert all(torch.equal(a, b) for a, b in zip(outs, eager[i]))
        assert all(torch.equal(a, b) for a, b in zip(between, eager[(i + 1) % 3]))
