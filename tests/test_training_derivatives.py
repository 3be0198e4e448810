"""Derivatives that the routing, sequence log-probability and preference operators do
not have: forward mode and second order are refused, never answered with a wrong value."""

import pytest
import torch
import torch.autograd.forward_ad as fw

import dot_amd

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def operators(dev):
    """name -> (function of the differentiable input, that input)."""
    gen = torch.Generator().manual_seed(0)
    make = lambda *s: torch.randn(*s, generator=gen).to(dev)  # noqa: E731
    experts = torch.randint(0, 8, (2, 5, 2), generator=gen).to(dev)
    tokens = torch.randint(0, 11, (4, 6), generator=gen).to(dev)
    ratio, plan = make(8), make(3, 5).abs()
    return {
        "weights": (lambda x: dot_amd.topk_routing(x, 2).weights, make(2, 5, 8)),
        "weights of one row set": (lambda x: dot_amd.topk_routing(x, 2, scoring="sigmoid", normalize=True).weights, make(5, 8)),
        "routing loss": (lambda x: dot_amd.topk_routing(x, 2).balance_loss, make(2, 5, 8)),
        "balance_loss": (lambda x: dot_amd.balance_loss(x, experts).loss, make(2, 5, 8)),
        "sequence_logp": (lambda x: dot_amd.sequence_logp(x, tokens), make(4, 6, 11)),
        "sequence_logp per token": (lambda x: dot_amd.sequence_logp(x, tokens, reduction="none"), make(4, 6, 11)),
        "pairs": (lambda x: dot_amd.preference_loss(x), ratio),
        "plan, ratios": (lambda x: dot_amd.preference_loss(x, plan=plan, loss_type="square"), ratio),
        "plan": (lambda x: dot_amd.preference_loss(ratio, plan=x), plan),
    }


NAMES = list(operators("cpu"))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(dev, name):
    f, x = operators(dev)[name]
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(fw.make_dual(x, torch.ones_like(x)))
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            f(fw.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="forward-mode|functorch"):
        torch.func.jvp(f, (x,), (torch.ones_like(x),))
    with fw.dual_level(), fw._set_fwd_grad_enabled(False):  # nothing is to be followed
        assert torch.equal(f(fw.make_dual(x, torch.ones_like(x))), f(x))


@pytest.mark.parametrize("dev", DEVICES)
def test_constants_may_have_tangents(dev):
    """The bias of a selection and the reference's log-probabilities are constants of every derivative."""
    gen = torch.Generator().manual_seed(1)
    x, bias = torch.randn(3, 8, generator=gen).to(dev), torch.randn(8, generator=gen).to(dev)
    tokens, ref = torch.randint(0, 8, (3,), generator=gen).to(dev), torch.randn(3, generator=gen).to(dev)
    with fw.dual_level():
        r = dot_amd.topk_routing(x, 2, bias=fw.make_dual(bias, torch.ones_like(bias)))
        out = dot_amd.sequence_logp(x, tokens, ref_logp=fw.make_dual(ref, torch.ones_like(ref)))
        assert fw.unpack_dual(r.weights).tangent is None and fw.unpack_dual(out).tangent is None
    assert torch.equal(r.weights, dot_amd.topk_routing(x, 2, bias=bias).weights)
    assert torch.equal(out, dot_amd.sequence_logp(x, tokens, ref_logp=ref))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("upstream", ["constant", "differentiable"])
@pytest.mark.parametrize("name", NAMES)
def test_second_order_is_refused(dev, upstream, name):
    """A gradient that create_graph asks for can be used, but nothing flows through it unnoticed."""
    f, x = operators(dev)[name]
    x.requires_grad_()
    out = f(x)
    loss = out.sum() if upstream == "constant" else (out * out).sum()
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    assert g.requires_grad
    (plain,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert not plain.requires_grad and torch.equal(g, plain)
    for total in (g.sum(), loss + (g**2).sum()):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(total, x, retain_graph=True)
    assert torch.equal(torch.autograd.grad(loss, x, retain_graph=True)[0], plain)
    up = torch.ones_like(out).requires_grad_()  # nor to the upstream gradient, in which g is linear
    (g,) = torch.autograd.grad(out, x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum(), up)


@pytest.mark.parametrize("dev", DEVICES)
def test_second_order_of_both_inputs_is_refused(dev):
    gen = torch.Generator().manual_seed(2)
    ratio = torch.randn(8, generator=gen).to(dev).requires_grad_()
    plan = torch.rand(3, 5, generator=gen).to(dev).requires_grad_()
    loss = dot_amd.preference_loss(ratio, plan=plan).sum()
    for g in torch.autograd.grad(loss, [ratio, plan], create_graph=True):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(g.sum(), [ratio, plan], retain_graph=True, allow_unused=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.functional.hessian(lambda r: dot_amd.preference_loss(r).sum(), ratio.detach())
    # leaves take the gradient of a graph that is kept
    loss.backward(create_graph=True)
    assert ratio.grad.requires_grad and plan.grad.requires_grad
    ratio.grad = plan.grad = None
