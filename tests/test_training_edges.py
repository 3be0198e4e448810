"""The routing, sequence log-probability and preference operators where their
rules decide: rows of masses too small to count, and the rules that the device
implementations share."""

import numpy as np
import pytest
import torch

import dot_amd
from conftest import rel_err
from oracle import training as oracle

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TOL = 1e-6  # results in fp32 of sums in 64 bits


def small_rows(scoring):
    """Scores (1, 6, 8) with rows whose masses, or whose two largest masses, sum to less than the
    smallest normal fp32 (1.2e-38), between ordinary ones."""
    rng = np.random.default_rng(0)
    if scoring == "plan":
        s = rng.random((1, 6, 8)) + 0.1
        s[0, 1] = 1e-42
        s[0, 2] = 1e-39 * np.arange(1, 9)    # 3.6e-38 in all, 1.5e-38 in the largest two
        s[0, 3] = 1e-40 * np.arange(1, 9)    # 3.6e-39 in all
        s[0, 4] = 0.0
    else:
        s = rng.standard_normal((1, 6, 8))
        s[0, 1] = -95.0
        s[0, 2] = -86.0 - np.arange(8)       # 4.5e-38, 1.6e-38, the others none
        s[0, 3] = -90.0
        s[0, 4] = -1e4
    return s.astype(np.float32)


@pytest.mark.parametrize("scoring", ["plan", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_masses_below_the_smallest_normal_count_as_none(scoring, normalize):
    s = small_rows(scoring)
    x = torch.as_tensor(s).requires_grad_()
    r = dot_amd.topk_routing(x, 2, scoring=scoring, normalize=normalize)
    o = oracle.route(s, 2, scoring, normalize)
    assert np.array_equal(r.experts.numpy(), o["experts"])
    assert rel_err(r.weights, o["weights"]) < TOL and rel_err(r.balance_loss, o["loss"]) < TOL
    none = [1, 3, 4]
    if normalize:
        assert (r.weights[0, none] == 0).all()
        assert rel_err(r.weights[0, [0, 2, 5]].sum(-1), torch.ones(3)) < TOL
    rng = np.random.default_rng(1)
    dw, dl = rng.standard_normal(o["weights"].shape).astype(np.float32), np.ones(1, np.float32)
    (g,) = torch.autograd.grad([r.weights, r.balance_loss], [x], [torch.as_tensor(dw), torch.as_tensor(dl)])
    og = oracle.route_grad(s, 2, o, scoring, normalize, None, dw, dl)
    assert np.isfinite(og).all() and torch.isfinite(g).all()
    rows = [0, 5]  # row 2's reciprocal mass is beyond the others'
    assert rel_err(g[0, rows], og[0, rows]) < TOL and rel_err(g[0, 2], og[0, 2]) < TOL
    # subnormal results are multiples of 2^-149: off by 2^-150, whatever their size
    assert (np.abs(g[0, none].numpy().astype(np.float64) - og[0, none]) <= TOL * np.abs(og[0, none]).max() + 2.0**-150).all()
    if normalize:
        assert (g[0, none] == 0).all()
    # such rows have no share in the loss, whatever they are assigned
    q = dot_amd.balance_loss(x[:, none], torch.zeros(1, 3, 1, dtype=torch.int32), scoring=scoring)
    assert q.loss.tolist() == [0.0] and q.counts[0].tolist() == [3] + [0] * 7
    assert (torch.autograd.grad(q.loss.sum(), x)[0] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bias_on_the_masses(dev, normalize, dtype):
    """A bias is added to the scores: to the logits with scoring="sigmoid", to sigmoid(logit) where the masses are
    given.  Weights and gradients are those of the sigmoid router's definition in 64 bits; fp32 operations in a chain
    of about ten (logistic function, shares, quotient, slope), 1e-5 of the largest value, and half a step of the type."""
    gen = torch.Generator().manual_seed(3)
    B, N, E, k = 2, 60, 64, 8
    logits = torch.randn(B, N, E, generator=gen).to(dtype).to(dev).requires_grad_()
    bias = (0.2 * torch.randn(E, generator=gen)).to(dev)
    q = torch.sigmoid(logits.float())
    r = dot_amd.topk_routing(q, k, scoring="plan", bias=bias, normalize=normalize)
    order = torch.argsort(-(q.detach() + bias), dim=-1, stable=True)[..., :k]  # q + bias, equal ones by the lowest index
    assert torch.equal(r.experts.long(), order)
    raw = dot_amd.topk_routing(logits.detach(), k, scoring="sigmoid", bias=bias)
    assert torch.equal(raw.experts.long(), torch.argsort(-(logits.detach().float() + bias), dim=-1, stable=True)[..., :k])
    assert not torch.equal(raw.experts.long().sort(-1).values, order.sort(-1).values)

    x = logits.detach().double().requires_grad_()
    s = torch.sigmoid(x)
    w = s.gather(-1, order)
    w = w / w.sum(-1, keepdim=True) if normalize else w
    counts = torch.stack([torch.bincount(t.reshape(-1), minlength=E) for t in order])
    loss = E * (counts / (k * N) * (s / s.sum(-1, keepdim=True)).mean(1)).sum(-1)
    assert torch.equal(r.counts.long(), counts)
    assert rel_err(r.weights, w) < 1e-5 and rel_err(r.balance_loss, loss) < 1e-5
    dw, dl = torch.randn(B, N, k, generator=gen).to(dev), torch.rand(B, generator=gen).to(dev)
    (g,) = torch.autograd.grad([r.weights, r.balance_loss], [logits], [dw, dl])
    (want,) = torch.autograd.grad([w, loss], [x], [dw.double(), dl.double()])
    assert rel_err(g.float(), want) < 1e-5 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
