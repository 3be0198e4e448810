"""CPU: the routing, sequence log-probability and preference operators — the
oracle's gradients against central differences, the CPU implementations against
the oracle, refusals before any kernel, and the C ABI's checks."""

import ctypes
import os

import numpy as np
import pytest
import torch

import dot
import dot_amd
from conftest import ROOT, rel_err
from oracle import training as oracle

TOL = 1e-6  # results in fp32 of sums in 64 bits


def differences(f, x, h=1e-5):
    """Central differences of a scalar function of an array."""
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        lo, hi = x.copy(), x.copy()
        lo[i] -= h
        hi[i] += h
        g[i] = (f(hi) - f(lo)) / (2 * h)
    return g


# fp32 scores on a grid of 2^-12 with a step of 2^-10: the oracle's keys are those of fp32
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "plan"])
@pytest.mark.parametrize("normalize", [False, True])
def test_oracle_routing_gradient(scoring, normalize):
    rng = np.random.default_rng(0)
    s = np.round(rng.standard_normal((2, 4, 5)) * 4096) / 4096
    if scoring == "plan":
        s = np.abs(s) + 0.25
    mask = np.array([[1, 1, 0, 1], [1, 0, 1, 1]], bool)
    dw, dl = rng.standard_normal((2, 4, 2)), rng.standard_normal(2)

    def total(x):
        o = oracle.route(x, 2, scoring, normalize, mask=mask)
        return (o["weights"] * dw).sum() + (o["loss"] * dl).sum()

    fwd = oracle.route(s, 2, scoring, normalize, mask=mask)
    g = oracle.route_grad(s, 2, fwd, scoring, normalize, mask, dw, dl)
    # h^2 / 6 of the third derivative: below 2^-20 of values of order 1
    assert np.abs(g - differences(total, s, h=2.0**-10)).max() < 2e-6


@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
def test_oracle_sequence_gradient(reduction):
    rng = np.random.default_rng(1)
    x, tokens = rng.standard_normal((2, 3, 6)), rng.integers(0, 6, (2, 3))
    tokens[0, 0] = -100
    mask = np.array([[1, 1, 1], [0, 1, 1]], bool)
    up = rng.standard_normal((2, 3) if reduction == "none" else 2)
    _, p, weight = oracle.sequence_logp(x, tokens, mask=mask, tau=0.7, reduction=reduction)
    g = oracle.sequence_logp_grad(p, weight, tokens, up, 0.7)
    d = differences(lambda z: (oracle.sequence_logp(z, tokens, mask=mask, tau=0.7, reduction=reduction)[0] * up).sum(), x)
    assert np.abs(g - d).max() < 1e-8


@pytest.mark.parametrize("loss_type,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.3), ("hinge", 0.0), ("square", 0.0)])
@pytest.mark.parametrize("coupled", [False, True])
def test_oracle_preference_gradient(loss_type, smoothing, coupled):
    rng = np.random.default_rng(2)
    r = 3 * rng.standard_normal(8)
    plan = rng.random((3, 5)) if coupled else None
    up = rng.random(3 if coupled else 4)
    _, gr, gp = oracle.preference(r, plan, 0.4, loss_type, smoothing, up)
    f = lambda a, b: (oracle.preference(a, b, 0.4, loss_type, smoothing)[0] * up).sum()  # noqa: E731
    assert np.abs(gr - differences(lambda z: f(z, plan), r)).max() < 1e-7
    if coupled:
        assert np.abs(gp - differences(lambda z: f(r, z), plan)).max() < 1e-7


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid", "plan"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_cpu_routing(scoring, normalize, dtype):
    rng = np.random.default_rng(3)
    s = rng.standard_normal((2, 9, 12))
    s = torch.as_tensor(np.abs(s) if scoring == "plan" else s).to(dtype)
    s[0, 0] = -float("inf")
    s[0, 1, 2:] = -float("inf")
    bias = rng.standard_normal(12).astype(np.float32)
    mask = rng.random((2, 9)) < 0.8
    mask[0, :2] = True
    s[~torch.as_tensor(mask)] = float("nan")
    x = s.clone().requires_grad_()
    r = dot_amd.topk_routing(x, 3, scoring=scoring, normalize=normalize, bias=torch.as_tensor(bias),
                             mask=torch.as_tensor(mask))
    o = oracle.route(s.float().numpy(), 3, scoring, normalize, bias, mask)
    assert np.array_equal(r.experts.numpy(), o["experts"]) and np.array_equal(r.counts.numpy(), o["counts"])
    assert rel_err(r.weights, o["weights"]) < TOL and rel_err(r.balance_loss, o["loss"]) < TOL
    dw, dl = rng.standard_normal(o["weights"].shape).astype(np.float32), rng.random(2).astype(np.float32)
    (g,) = torch.autograd.grad([r.weights, r.balance_loss], [x], [torch.as_tensor(dw), torch.as_tensor(dl)])
    og = oracle.route_grad(s.float().numpy(), 3, o, scoring, normalize, mask, dw, dl)
    tol = TOL + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    assert g.dtype == dtype and rel_err(g.float(), og) < tol
    # given experts: the same counts and loss
    q = dot_amd.balance_loss(x, r.experts.long(), scoring=scoring, mask=torch.as_tensor(mask))
    assert torch.equal(q.counts, r.counts) and torch.equal(q.loss, r.balance_loss)


def test_cpu_routing_ties_and_slots():
    s = torch.tensor([[0.0, -0.0, 0.0, 1.0], [2.0, 2.0, 2.0, 2.0]])
    r = dot_amd.topk_routing(s, 3)
    assert r.experts.tolist() == [[3, 0, 1], [0, 1, 2]] and r.counts.tolist() == [2, 2, 1, 1]
    q = dot_amd.balance_loss(s, torch.tensor([[0, -1], [3, 3]]))
    assert q.counts.tolist() == [1, 0, 0, 2]


@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cpu_sequence_logp(reduction, dtype):
    rng = np.random.default_rng(4)
    x = torch.as_tensor(rng.standard_normal((2, 5, 30)).astype(np.float32)).to(dtype).requires_grad_()
    tokens = rng.integers(0, 30, (2, 5))
    tokens[0, 1] = -100
    mask = rng.random((2, 5)) < 0.7
    ref = rng.standard_normal((2, 5))
    out = dot_amd.sequence_logp(x, torch.as_tensor(tokens), ref_logp=torch.as_tensor(ref), mask=torch.as_tensor(mask),
                                tau=0.8, reduction=reduction)
    o, p, w = oracle.sequence_logp(x.detach().float().numpy(), tokens, ref, mask, 0.8, reduction)
    assert rel_err(out, o) < TOL
    up = rng.standard_normal(o.shape).astype(np.float32)
    (g,) = torch.autograd.grad([out], [x], [torch.as_tensor(up)])
    tol = TOL + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    assert rel_err(g.float(), oracle.sequence_logp_grad(p, w, tokens, up, 0.8)) < tol


@pytest.mark.parametrize("loss_type,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.3), ("hinge", 0.0), ("square", 0.0)])
def test_cpu_preference(loss_type, smoothing):
    rng = np.random.default_rng(5)
    ratio = (4 * rng.standard_normal(12)).astype(np.float32)
    for plan in (None, rng.random((5, 7)).astype(np.float32)):
        r = torch.as_tensor(ratio).requires_grad_()
        pl = None if plan is None else torch.as_tensor(plan).requires_grad_()
        loss = dot_amd.preference_loss(r, plan=pl, beta=0.3, loss_type=loss_type, label_smoothing=smoothing)
        o, gr, gp = oracle.preference(ratio, plan, 0.3, loss_type, smoothing)
        grads = torch.autograd.grad(loss.sum(), [r] + ([] if pl is None else [pl]))
        assert rel_err(loss, o) < TOL and rel_err(grads[0], gr) < TOL
        assert pl is None or rel_err(grads[1], gp) < TOL


def test_cpu_pairs_left_out():
    ratio = torch.tensor([1.0, float("nan"), 0.5, float("-inf")], requires_grad=True)
    plan = torch.tensor([[0.5, 0.0], [0.0, 0.0]], requires_grad=True)
    loss = dot_amd.preference_loss(ratio, plan=plan)
    g, gp = torch.autograd.grad(loss.sum(), [ratio, plan])
    assert torch.isfinite(loss).all() and loss[1] == 0 and torch.isfinite(g).all() and torch.isfinite(gp).all()


def test_cpu_empty():
    r = dot_amd.topk_routing(torch.zeros(2, 0, 4), 2)
    assert r.weights.shape == (2, 0, 2) and (r.balance_loss == 0).all()
    assert dot_amd.sequence_logp(torch.zeros(2, 0, 4), torch.zeros(2, 0, dtype=torch.long)).tolist() == [0, 0]
    assert dot_amd.preference_loss(torch.zeros(0)).shape == (0,)


def test_modules_and_names():
    x = torch.randn(2, 6, 8)
    a, b = dot.TopKRouting(2, normalize=True)(x), dot.topk_routing(x, 2, normalize=True)
    assert torch.equal(a.weights, b.weights)
    assert torch.equal(dot.BalanceLoss("sigmoid")(x, b.experts).loss, dot.balance_loss(x, b.experts, scoring="sigmoid").loss)
    t = torch.randint(0, 8, (2, 6))
    assert torch.equal(dot.SequenceLogp(0.5, "mean")(x, t), dot.sequence_logp(x, t, tau=0.5, reduction="mean"))
    r = torch.randn(4)
    assert torch.equal(dot.PreferenceLoss(0.3, "hinge")(r), dot.preference_loss(r, beta=0.3, loss_type="hinge"))
    import importlib
    assert importlib.import_module("dot.routing").topk_routing is dot_amd.topk_routing
    assert importlib.import_module("dot.preference").preference_loss is dot_amd.preference_loss


def test_second_derivatives_are_refused():
    x = torch.randn(1, 3, 4, requires_grad=True)
    (g,) = torch.autograd.grad(dot_amd.topk_routing(x, 1).balance_loss.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_refusals():
    x = torch.randn(2, 5, 8)
    bad = [
        (lambda: dot.topk_routing(x, 0), "k must be"), (lambda: dot.topk_routing(x, 9), "k must be"),
        (lambda: dot.topk_routing(x, 2.0), "k must be"), (lambda: dot.topk_routing(x, True), "k must be"),
        (lambda: dot.topk_routing(torch.randn(1, 2, 100), 65), "k must be"),
        (lambda: dot.topk_routing(x, 2, scoring="tanh"), "scoring"),
        (lambda: dot.topk_routing(x.double(), 2), "float32"), (lambda: dot.topk_routing(x[0, 0], 2), "shape"),
        (lambda: dot.topk_routing(torch.zeros(1, 1, 4097), 2), "experts are supported"),
        (lambda: dot.topk_routing(torch.zeros(1, 1, 0), 1), "experts are supported"),
        (lambda: dot.topk_routing(x, 2, bias=torch.zeros(7)), "bias"),
        (lambda: dot.topk_routing(x, 2, bias=torch.zeros(8, dtype=torch.int32)), "bias"),
        (lambda: dot.topk_routing(x, 2, mask=torch.ones(2, 5)), "mask"),
        (lambda: dot.topk_routing(x, 2, mask=torch.ones(2, 6, dtype=torch.bool)), "mask"),
        (lambda: dot.balance_loss(x, torch.zeros(2, 5, 2)), "int32 or int64"),
        (lambda: dot.balance_loss(x, torch.zeros(2, 4, 2, dtype=torch.int32)), "experts must have shape"),
        (lambda: dot.balance_loss(x, torch.zeros(5, 2, dtype=torch.int32)), "experts must have shape"),
        (lambda: dot.balance_loss(x, torch.zeros(2, 5, 65, dtype=torch.int32)), "per token"),
        (lambda: dot.balance_loss(x, torch.zeros(2, 5, 0, dtype=torch.int32)), "per token"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 5)), "tokens"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 4, dtype=torch.long)), "tokens"),
        (lambda: dot.sequence_logp(x.double(), torch.zeros(2, 5, dtype=torch.long)), "float32"),
        (lambda: dot.sequence_logp(torch.zeros(2, 5, 0), torch.zeros(2, 5, dtype=torch.long)), "V >= 1"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 5, dtype=torch.long), tau=0.0), "tau"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 5, dtype=torch.long), tau=float("nan")), "tau"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 5, dtype=torch.long), reduction="max"), "reduction"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 5, dtype=torch.long), mask=torch.ones(2, 5)), "mask"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 5, dtype=torch.long), ref_logp=torch.zeros(3)), "ref_logp"),
        (lambda: dot.sequence_logp(x, torch.zeros(2, 5, dtype=torch.long), ref_logp=torch.zeros(2), reduction="none"),
         "per position"),
        (lambda: dot.preference_loss(torch.zeros(3)), "even"), (lambda: dot.preference_loss(torch.zeros(2, 2)), "vector"),
        (lambda: dot.preference_loss(torch.zeros(4, dtype=torch.int32)), "vector"),
        (lambda: dot.preference_loss(torch.zeros(4), plan=torch.zeros(3, 3)), "plan"),
        (lambda: dot.preference_loss(torch.zeros(4), plan=torch.zeros(4)), "plan"),
        (lambda: dot.preference_loss(torch.zeros(4), beta=0.0), "beta"),
        (lambda: dot.preference_loss(torch.zeros(4), loss_type="log"), "loss_type"),
        (lambda: dot.preference_loss(torch.zeros(4), label_smoothing=1.0), "label_smoothing"),
        (lambda: dot.preference_loss(torch.zeros(4), loss_type="hinge", label_smoothing=0.1), "label_smoothing"),
    ]
    for f, text in bad:
        with pytest.raises(ValueError, match=text):
            f()


# ---------------------------------------------------------------------------
# C ABI: bad arguments are refused on the host
# ---------------------------------------------------------------------------
@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(ROOT, "dot_amd", "libdot_amd.so"))
    lib.dot_last_error.restype = ctypes.c_char_p
    for name in ("dot_routing_forward_workspace_bytes", "dot_seqlogp_forward_workspace_bytes",
                 "dot_preference_backward_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_size_t
    return lib


P, I, I64, F, D, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_double, ctypes.c_size_t


def struct(*fields):
    return type("Args", (ctypes.Structure,), {"_fields_": list(fields)})


RoutingFwd = struct(("scores", P), ("dtype", I), ("stride_b", I64), ("stride_n", I64), ("B", I), ("N", I), ("E", I),
                    ("k", I), ("scoring", I), ("normalize", I), ("bias", P), ("mask", P), ("given", P),
                    ("given_is_int64", I), ("weights", P), ("experts", P), ("counts", P), ("tokens", P), ("loss", P),
                    ("workspace", P), ("workspace_bytes", Z))
RoutingBwd = struct(("scores", P), ("dtype", I), ("stride_b", I64), ("stride_n", I64), ("B", I), ("N", I), ("E", I),
                    ("k", I), ("scoring", I), ("normalize", I), ("mask", P), ("counts", P), ("tokens", P),
                    ("grad_loss", P), ("grad_loss_scalar", I), ("weights", P), ("experts", P), ("grad_weights", P),
                    ("grad_scores", P))
SeqFwd = struct(("logits", P), ("dtype", I), ("stride_b", I64), ("stride_s", I64), ("B", I), ("S", I), ("V", I),
                ("tokens", P), ("tokens_are_int64", I), ("mask", P), ("ref", P), ("ref_is_f64", I),
                ("ref_per_token", I), ("tau", D), ("reduction", I), ("out", P), ("row_stats", P), ("weight", P),
                ("workspace", P), ("workspace_bytes", Z))
PrefFwd = struct(("ratio", P), ("plan", P), ("P", I), ("Q", I), ("loss_type", I), ("beta", F), ("smoothing", F),
                 ("loss", P))
PrefBwd = struct(("ratio", P), ("plan", P), ("P", I), ("Q", I), ("loss_type", I), ("beta", F), ("smoothing", F),
                 ("grad_loss", P), ("grad_loss_scalar", I), ("grad_ratio", P), ("grad_plan", P), ("workspace", P),
                 ("workspace_bytes", Z))
INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 3


def refused(lib, name, code, text, args):
    assert getattr(lib, name)(None if args is None else ctypes.byref(args), None) == code
    assert text in lib.dot_last_error().decode()


def test_c_abi_refusals(lib):
    some = 256  # an address that is never read: every call here is refused before a launch
    ok = dict(scores=some, B=2, N=4, E=8, k=2, stride_b=32, stride_n=8, weights=some, experts=some, counts=some,
              tokens=some, loss=some)
    f = "dot_routing_forward"
    refused(lib, f, INVALID, "NULL", None)
    refused(lib, f, INVALID, "dtype", RoutingFwd(**{**ok, "dtype": 7}))
    refused(lib, f, INVALID, "E must be", RoutingFwd(**{**ok, "E": 0}))
    refused(lib, f, UNSUPPORTED, "MAX_EXPERTS", RoutingFwd(**{**ok, "E": 4097}))
    refused(lib, f, INVALID, "at most E", RoutingFwd(**{**ok, "k": 9}))
    refused(lib, f, UNSUPPORTED, "MAX_K", RoutingFwd(**{**ok, "k": 65}))
    refused(lib, f, INVALID, "scoring", RoutingFwd(**{**ok, "scoring": 3}))
    refused(lib, f, INVALID, "non-NULL", RoutingFwd(**{**ok, "loss": None}))
    refused(lib, f, INVALID, "non-NULL", RoutingFwd(**{**ok, "experts": None}))
    many = {**ok, "N": 100000}  # few tokens are joined in one workgroup and need none
    refused(lib, f, WORKSPACE, "workspace", RoutingFwd(**many))
    need = lib.dot_routing_forward_workspace_bytes(2, 100000, 8)
    assert need > 0 and lib.dot_routing_forward_workspace_bytes(-1, 4, 8) == 0
    refused(lib, f, WORKSPACE, "workspace", RoutingFwd(**many, workspace=some, workspace_bytes=need - 1))
    b = dict(scores=some, B=2, N=4, E=8, k=2, counts=some, tokens=some, grad_loss=some, grad_scores=some)
    f = "dot_routing_backward"
    refused(lib, f, INVALID, "non-NULL", RoutingBwd(**{**b, "grad_scores": None}))
    refused(lib, f, INVALID, "counts", RoutingBwd(**{**b, "counts": None}))
    refused(lib, f, INVALID, "tokens", RoutingBwd(**{**b, "tokens": None, "mask": some}))
    refused(lib, f, INVALID, "weights", RoutingBwd(**{**b, "grad_weights": some}))

    s = dict(logits=some, B=2, S=3, V=16, tokens=some, tau=1.0, reduction=1, out=some)
    f = "dot_seqlogp_forward"
    refused(lib, f, INVALID, "tau", SeqFwd(**{**s, "tau": 0.0}))
    refused(lib, f, UNSUPPORTED, "tau", SeqFwd(**{**s, "tau": 1e-30}))
    refused(lib, f, INVALID, "V must", SeqFwd(**{**s, "V": 0}))
    refused(lib, f, UNSUPPORTED, "2^23", SeqFwd(**{**s, "B": 4096, "S": 4096}))
    refused(lib, f, INVALID, "reduction", SeqFwd(**{**s, "reduction": 5}))
    refused(lib, f, INVALID, "per sequence", SeqFwd(**{**s, "reduction": 0, "ref": some}))
    refused(lib, f, INVALID, "non-NULL", SeqFwd(**{**s, "tokens": None}))
    refused(lib, f, WORKSPACE, "workspace", SeqFwd(**s))

    p = dict(ratio=some, P=4, Q=4, beta=1.0, loss=some)
    f = "dot_preference_forward"
    refused(lib, f, INVALID, "P = Q", PrefFwd(**{**p, "Q": 5}))
    refused(lib, f, INVALID, "beta", PrefFwd(**{**p, "beta": -1.0}))
    refused(lib, f, INVALID, "smoothing", PrefFwd(**{**p, "smoothing": 1.0}))
    refused(lib, f, INVALID, "smoothing", PrefFwd(**{**p, "smoothing": 0.5, "loss_type": 1}))
    refused(lib, f, INVALID, "loss_type", PrefFwd(**{**p, "loss_type": 9}))
    refused(lib, f, UNSUPPORTED, "2^22", PrefFwd(**{**p, "P": 1 << 23, "Q": 1 << 23}))
    q = dict(ratio=some, plan=some, P=4, Q=6, beta=1.0, grad_loss=some, grad_ratio=some)
    refused(lib, "dot_preference_backward", WORKSPACE, "workspace", PrefBwd(**q))
    refused(lib, "dot_preference_backward", INVALID, "non-NULL", PrefBwd(**{**q, "grad_loss": None}))
