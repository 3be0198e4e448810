"""Top log-probabilities, distillation and beam search where their rules decide; tolerances in generation_cases.py."""

import ctypes
import os

import numpy as np
import pytest
import torch

import dot_amd
from conftest import ROOT
from generation_cases import DTYPES, check_beam, check_distill, check_top, logits_of, teacher_of
from oracle import generation as oracle

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def distill(dev, logits, logp, tokens, **kw):
    """check_distill of teacher tensors as they are given; -> (loss, gradient) on the CPU."""
    tk = torch.as_tensor(tokens).to(dev)

    def call(x, mask, **kw):
        mask = None if mask is None else torch.as_tensor(mask).to(dev)
        return dot_amd.distill_loss(x, logp.to(dev), tk, mask=mask, **kw)

    out, g = check_distill(call, logits, logp.float().numpy(), tokens, x=logits.to(dev), **kw)
    return out.cpu(), g.cpu().double()


# ---------------------------------------------------------------------------
# Teachers whose probabilities sum to more than 1
# ---------------------------------------------------------------------------
def test_gradient_of_masses_above_one_by_differences():
    """The loss written out: there is no rest, and the probabilities that are named are taken as they are."""
    rng = np.random.default_rng(0)
    tau, p, at = 0.8, np.array([0.9, 0.6]), [1, 4]
    logp = np.log(p).astype(np.float32)[None, None]
    p = np.exp(logp[0, 0].astype(np.float64))
    x = rng.standard_normal((1, 1, 6))

    def loss(x):
        z = x[0, 0] / tau
        return (p * (np.log(p) - (z - np.log(np.exp(z).sum()))[at])).sum()

    want = np.zeros(6)
    for v in range(6):
        d = np.zeros_like(x)
        d[0, 0, v] = 1e-5
        want[v] = (loss(x + d) - loss(x - d)) / 2e-5  # off by h^2 / 6 of a third derivative of order 1, and 1e-16 / h
    value, parts = oracle.distill(x, logp, np.array([[at]]), tau=tau, reduction="sum")
    g = oracle.distill_grad(x.shape, parts, np.ones(1), tau)[0, 0]
    assert abs(value[0] - loss(x)) < 1e-12 and np.abs(g - want).max() < 1e-8
    leaf = torch.as_tensor(x.astype(np.float32)).requires_grad_()
    out = dot_amd.distill_loss(leaf, torch.as_tensor(logp), torch.as_tensor([[at]]), tau=tau, reduction="sum")
    (g,) = torch.autograd.grad(out.sum(), leaf)
    # the logits in fp32 move the gradient by 2^-24 of them, and it is rounded once
    assert np.abs(g[0, 0].numpy() - want).max() < 1e-6


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("kept", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V,k", [(6, 2), (300, 40), (4000, 64), (70000, 64), (300000, 200)])
def test_masses_above_one(dev, kept, V, k):
    """Log-probabilities kept in 16 bits, and ones that are too large by 0.05: the gradient sums to 0 over a row."""
    print(f"[edges] mass {dev} {kept} V={V} k={k}", flush=True)
    rng = np.random.default_rng(V)
    logits = logits_of(rng, (2, 6, V), torch.float32)
    logp, tokens = teacher_of(rng, logits, k, tau=0.7, noise=0.3)
    logp = torch.as_tensor(logp)
    logp[0] = torch.where(logp[0] > -1, logp[0] + 0.05, logp[0]).clamp(max=-1e-3)
    logp = logp.to(kept)
    mass = logp.double().exp().sum(-1)
    assert (mass > 1.001).any() and mass.max() < 2
    for reduction in ("mean", "none"):
        _, g = distill(dev, logits, logp, tokens, tau=0.7, reduction=reduction)
        # each entry to the bound above, of which the row's have 3 SUM M / tau and 1e-5 of themselves
        assert (g.sum(-1).abs() <= (9e-6 * 2 + 2e-5) * g.abs().sum(-1) + 2e-5).all()
    distill(dev, logits, logp, tokens, tau=0.7, direction="reverse")
    distill(dev, logits, logp, tokens, tau=0.7, rest="none")


# ---------------------------------------------------------------------------
# What rounding leaves of a teacher's rest
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("offset", [0.0, 50.0, 500.0, -1000.0])
@pytest.mark.parametrize("tau", [0.9, 1.3])
def test_rest_of_a_list_of_a_whole_vocabulary(dev, offset, tau):
    """top_logp rounds scaled logits to fp32: log-probabilities are off by 2^-23 |x| / tau together, and what they
    leave of 1 with them (1.3e-4 at |x| / tau = 1112).  It is not held against a student that has no other token."""
    rng = np.random.default_rng(11)
    few = torch.as_tensor((3 * rng.standard_normal((1, 64, 200)) + offset).astype(np.float32))
    wide = torch.full((1, 64, 5000), -float("inf"))
    wide[..., 7:2007:10] = few  # the same tokens of a vocabulary of which the others are not allowed
    for x in (few, wide):
        t = dot_amd.top_logp(x.to(dev), 200, tau=tau)
        rest = 1 - t.logp.double().exp().sum(-1)
        assert rest.abs().max() < 2.0**-12 and (offset == 0 or rest.max() > 2.0**-20)
        out, g = distill(dev, x, t.logp.cpu(), t.tokens.cpu().numpy(), tau=tau, reduction="none")
        # the student's own: the divergence is what the lists are off by
        assert torch.isfinite(out).all() and out.abs().max() < 2.0**-12 and g.abs().max() < 2.0**-12
    # a rest that is none of rounding has no place
    less = t.logp.cpu() - 2.0**-11
    out = dot_amd.distill_loss(wide.to(dev), less.to(dev), t.tokens, tau=tau, reduction="none")
    assert (out == float("inf")).all()


# ---------------------------------------------------------------------------
# Rows that begin with tokens that are not allowed
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [3000, 32768, 100003, 131072])
@pytest.mark.parametrize("offset", [-69.0, -40.0, 30.0, 150.0])
def test_banned_beginnings(dev, dtype, V, offset):
    """Blocks of -inf as long as what a workgroup's threads take at once, and logits far from 0 behind them: the many
    small terms of the sum count as where the logits lie around 0."""
    print(f"[edges] banned {dev} {dtype} V={V} {offset}", flush=True)
    rng = np.random.default_rng(V)
    x = rng.standard_normal((1, 4, V)) + offset - 20
    x[..., V // 2 + 5] = offset
    at = np.arange(V)
    long = 8 if dtype != "fp32" else 4
    for row, every in enumerate((16 * 256 * long, 4 * 256 * long, 1024 * 8, 1 << 30)):
        x[0, row, at % every < (256 * long if every < 1 << 30 else V // 3)] = -np.inf
    logits = torch.as_tensor(x.astype(np.float32)).to(DTYPES[dtype])
    for k in (1, 20, 100):
        check_top(dot_amd.top_logp(logits.to(dev), k), logits, k)
    scores = -np.arange(4.0)[None]
    r = dot_amd.beam_step(logits.to(dev), torch.as_tensor(scores.astype(np.float32)).to(dev), k=8)
    check_beam(r, logits, scores, 8)


# ---------------------------------------------------------------------------
# States in each other's gaps
# ---------------------------------------------------------------------------
def neighbours():
    """name -> (shape, views of it), with states of different sizes beside each other."""
    return {
        "widths": ((2, 4, 3, 8, 80), lambda t: [t[..., :64], t[..., 64:]]),
        "heads": ((2, 4, 8, 6, 16), lambda t: [t[:, :, :, :4], t[:, :, :, 4:]]),
        "lengths": ((2, 4, 3, 8, 16), lambda t: [t[:, :, :, :5], t[:, :, :, 5:]]),
        "outer": ((2, 4, 5, 8, 16), lambda t: [t[:, :, :2], t[:, :, 2:3], t[:, :, 3:]]),
        "tokens beside": ((2, 4, 3, 40), lambda t: [t[..., 8:], t[:, :, 0, 1], t[:, :, 1, :3]]),
        "positions first": ((6, 2, 4, 3, 20), lambda t: [t[..., :16].permute(1, 2, 0, 3, 4), t[..., 16:].permute(1, 2, 0, 3, 4)]),
        "layers": ((2, 4, 3, 2, 6, 24), lambda t: [v for i in range(3) for v in (t[:, :, i, 0, :, :16], t[:, :, i, 1])]),
    }


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("name", list(neighbours()))
def test_states_beside_each_other(dev, name):
    print(f"[edges] beside {dev} {name}", flush=True)
    shape, views = neighbours()[name]
    t = torch.arange(np.prod(shape), dtype=torch.float32).view(shape)
    beams = torch.as_tensor([[3, 0, 0, 7], [-1, 2, 1, 3]])
    want = t.clone()
    for v, old in zip(views(want), views(t)):
        v.copy_(torch.as_tensor(oracle.beam_reorder(old.numpy(), beams.tolist())))
    x = t.to(dev)
    dot_amd.beam_reorder(views(x), beams.to(dev))
    assert torch.equal(x.cpu(), want)


def test_states_that_meet_are_refused():
    beams = torch.as_tensor([[3, 0, 0, 7], [-1, 2, 1, 3]])
    for shape, views in (((2, 4, 3, 8, 80), lambda t: [t[..., :65], t[..., 64:]]),
                         ((2, 4, 8, 6, 16), lambda t: [t[:, :, :, :4], t[:, :, :, 3:]]),
                         ((2, 4, 3, 40), lambda t: [t, t[:, :, 2, :1]])):
        with pytest.raises(ValueError, match="share memory"):
            dot_amd.beam_reorder(views(torch.zeros(shape)), beams)
    # the beams themselves between the states' places, and in them
    arena = torch.zeros(80, dtype=torch.int64)
    state = arena.as_strided((2, 4, 4), (40, 6, 1))
    for at, ok in ((22, True), (32, True), (15, False), (33, False)):
        inside = arena[at : at + 8].view(2, 4)
        inside.copy_(beams)
        if ok:
            dot_amd.beam_reorder(state, inside)
        else:
            with pytest.raises(ValueError, match="share memory"):
                dot_amd.beam_reorder(state, inside)
        inside.zero_()


def test_meeting_states_by_their_bytes():
    """The check of random states against the sets of their bytes."""
    fields = [("data", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("sb", "sw", "so", "sp", "outer", "positions", "inner")]
    State = type("State", (ctypes.Structure,), {"_fields_": fields})
    P, I = ctypes.c_void_p, ctypes.c_int  # noqa: E741
    Args = type("Args", (ctypes.Structure,), {"_fields_": [("states", P), ("count", I), ("B", I), ("W", I), ("beams", P),
                                                           ("beams64", I), ("lengths", P), ("lengths64", I)]})
    check = ctypes.CDLL(os.path.join(ROOT, "dot_amd", "libdot_amd.so")).dot_beam_reorder_check
    rng = np.random.default_rng(0)

    def state_of(sizes, strides, at, inner):
        by = dict(zip(("sb", "sw", "so", "sp"), strides))
        return State(data=at, outer=sizes[2], positions=sizes[3], inner=inner, **{k: int(v) for k, v in by.items()})

    def bytes_of(sizes, strides, at, inner):
        grid = np.zeros(1, np.int64) + at
        for n, s in zip((*sizes, inner), (*strides, 1)):
            grid = (grid[:, None] + s * np.arange(n)).ravel()
        return set(grid.tolist())

    def nested(sizes, inner):
        """Strides in a random order, each past what the smaller ones reach."""
        strides, reach = np.zeros(4, np.int64), inner
        for d in rng.permutation(4):
            strides[d] = reach + rng.integers(0, 9)
            reach = strides[d] * (sizes[d] - 1) + reach
        return strides

    met = 0
    for trial in range(3000):
        sizes = rng.integers(1, 4, 4)
        inner = int(rng.integers(1, 5))
        strides = nested(sizes, inner + 3)
        other, other_inner = sizes.copy(), int(rng.integers(1, 5))
        other[2:] = rng.integers(1, 4, 2)
        same = rng.random() < 0.6 and all(other <= sizes)
        other_strides = strides if same else nested(other, other_inner)
        x, y = (sizes, strides, 4096, inner), (other, other_strides, 4096 + int(rng.integers(-30, 60)), other_inner)
        states = (State * 2)(state_of(*x), state_of(*y))
        args = Args(states=ctypes.addressof(states), count=2, B=int(sizes[0]), W=int(sizes[1]), beams=1 << 40)
        shared = bool(bytes_of(*x) & bytes_of(*y))
        met += shared
        assert check(ctypes.byref(args)) == (1 if shared else 0), (trial, x, y)
    assert 300 < met < 2700


# ---------------------------------------------------------------------------
# Temperatures that no float holds
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("sign", [1, -1])
def test_gradients_of_far_tokens_have_no_common_error(dev, sign):
    """log2(e) / tau as one float is off by up to 2^-24 of itself, and so are the exponents of all tokens at one
    distance, in one direction.

    Of 20000 tokens about 60 tau below the likeliest, the relative errors of fp32 gradients are those of the rounded
    exponents, of either sign (2^-18 ln 2 at most each: 3e-8 in the mean of all, six standard deviations 1e-7), and
    what they have in common: 4 roundings of the row's factor and 2^-23 of the exponential, 4e-7."""
    taus = np.linspace(0.5, 2, 4001)
    k = np.log2(np.e) / taus
    tau = float(taus[np.argmax(sign * (k.astype(np.float32) - k) / k)])
    rng = np.random.default_rng(5)
    x = np.full((1, 2, 20002), 0.0)
    x[..., 2:] = tau * (-60 + rng.random((1, 2, 20000)))
    logits = torch.as_tensor(x.astype(np.float32))
    logp, tokens = np.log(np.full((1, 2, 1), 0.5)).astype(np.float32), np.zeros((1, 2, 1), np.int64)
    for direction in ("forward", "reverse"):
        _, g = distill(dev, logits, torch.as_tensor(logp), tokens, tau=tau, direction=direction, reduction="none")
        _, parts = oracle.distill(logits.double().numpy(), logp, tokens, tau=tau, direction=direction, reduction="none")
        up = (0.5 + np.random.default_rng(0).random((1, 2))).astype(np.float32)  # as check_distill draws it
        want = oracle.distill_grad(logits.shape, parts, up, tau)[..., 2:]
        assert np.abs((g.numpy()[..., 2:] / want - 1).mean(-1)).max() < 5e-7


# ---------------------------------------------------------------------------
# Small and uneven rows
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_a_vocabulary_of_one(dev, dtype):
    rng = np.random.default_rng(6)
    logits = torch.as_tensor(rng.standard_normal((2, 128, 1)).astype(np.float32)).to(DTYPES[dtype])
    logits[1, 5] = -float("inf")
    check_top(dot_amd.top_logp(logits.to(dev), 1), logits, 1)
    scores = -np.sort(rng.random((2, 128)), 1)
    r = dot_amd.beam_step(logits.to(dev), torch.as_tensor(scores.astype(np.float32)).to(dev))
    check_beam(r, logits, scores, 128)
    logits = logits[:, 6:]  # a position without an allowed token has no divergence to compare
    logp, tokens = np.full((2, 122, 1), -0.25, np.float32), np.zeros((2, 122, 1), np.int64)
    for direction, rest in (("forward", "none"), ("reverse", "bucket")):
        distill(dev, logits, torch.as_tensor(logp), tokens, direction=direction, rest=rest)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("filler", ["-inf", "lowest", "low"])
@pytest.mark.parametrize("V", [5000, 40000])
def test_distillation_behind_a_filler(dev, dtype, V, filler):
    """Rows that begin with tokens that are not allowed, as long as a workgroup's first packs and longer."""
    print(f"[edges] filler {dev} {dtype} V={V} {filler}", flush=True)
    rng = np.random.default_rng(V)
    x = logits_of(rng, (1, 4, V), DTYPES[dtype])
    value = {"-inf": -float("inf"), "lowest": torch.finfo(x.dtype).min, "low": -1e4}[filler]
    logp, tokens = teacher_of(rng, x[..., V // 2 :], 30, tau=0.7)
    tokens = tokens + V // 2
    for row, n in enumerate((1, 4096, V // 2 - 1, V // 2)):
        x[0, row, :n] = value
    for direction, rest in (("forward", "bucket"), ("forward", "none"), ("reverse", "bucket")):
        out, g = distill(dev, x, torch.as_tensor(logp), tokens, tau=0.7, direction=direction, rest=rest, reduction="none")
        # where a named token is not allowed P log Q is -inf: 4096 tokens are more than half of 5000
        named = torch.as_tensor(np.take_along_axis(x.float().numpy(), tokens, -1))
        if filler == "-inf":
            assert torch.equal(torch.isinf(out), torch.isinf(named).any(-1) & (direction == "forward"))
        assert not torch.isnan(out).any() and torch.isfinite(g).all()
