"""Inputs and comparisons that the tests of the top log-probabilities, the distillation loss
and the beam search share.

Tolerances.  A sum s of V exponentials relative to the row's largest logit m: each term's
argument is off by 3 roundings of |x - m| / tau (difference, scale, product) and its
exponential by 2^-23, so s by 3 2^-24 E[(m - x) / tau] + 2^-23 of itself, E under the row's own
softmax, which is at most log V = 12: 2.3e-6; pairwise sums of 8 add 3 roundings, 1.8e-7.
So log s is off by SUM = 3e-6 at most.  top_logp and beam_step scale the logits in fp32
and then take their difference from the largest one: 2^-24 of both scaled logits, of the
difference, and 2^-24 of 1 / tau, which is 2^-24 of the difference again.
"""

import numpy as np
import torch

from oracle import generation as oracle

SUM = 3e-6
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def logits_of(rng, shape, dtype, spread=2.0):
    x = spread * rng.standard_normal(shape)
    for _ in range(3):  # some likelier tokens
        at = rng.integers(0, shape[-1], shape[:-1])
        np.put_along_axis(x, at[..., None], np.log(shape[-1]) + 5 * rng.random(shape[:-1])[..., None], -1)
    return torch.as_tensor(x.astype(np.float32)).to(dtype)


def array(t):
    return t.detach().cpu().double().numpy()


def share_error(x, beams, tokens, tau):
    """Error of (x_v - m) / tau for the entries (beam, token) of x (..., W, V); of no meaning in empty slots."""
    m = np.where(np.isfinite(x), x, -np.inf).max(-1, initial=-np.inf)
    m = np.take_along_axis(np.where(m == -np.inf, 0.0, m), np.maximum(beams, 0), -1)
    flat = x.reshape(*x.shape[:-2], -1)
    v = np.take_along_axis(flat, np.maximum(beams, 0) * x.shape[-1] + np.maximum(tokens, 0), -1)
    with np.errstate(invalid="ignore"):
        return 2.0**-24 * (np.abs(v) + np.abs(m) + 2 * np.abs(v - m)) / tau


def check_top(r, logits, k, tau=1.0, mask=None):
    """Tokens as they are, log-probabilities to the errors of the sum, of the share and half a step of fp32."""
    want, tokens = oracle.top_logp(array(logits), k, tau, mask)
    assert r.logp.dtype == torch.float32 and r.tokens.dtype == torch.int32
    assert r.logp.shape == want.shape and r.tokens.shape == want.shape
    assert np.array_equal(r.tokens.cpu().numpy(), tokens)
    got = array(r.logp)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    ok = np.isfinite(want)
    got, want, share = got[ok], want[ok], share_error(array(logits)[..., None, :], 0 * tokens, tokens, tau)[ok]
    assert (np.abs(got - want) <= SUM + share + 2.0**-24 * np.abs(want)).all(), np.abs(got - want).max()


def teacher_of(rng, logits, k, tau=1.0, noise=1.0):
    """Top k of a model near these logits: (logp float32, tokens)."""
    x = (array(logits) + noise * rng.standard_normal(logits.shape)) / tau
    lp = oracle.log_softmax(x)
    at = np.argsort(-lp, -1, kind="stable")[..., :k]
    return np.take_along_axis(lp, at, -1).astype(np.float32), at


def check_distill(call, logits, logp, tokens, mask=None, tau=1.0, direction="forward", rest="bucket",
                  reduction="mean", x=None, seed=0):
    """Loss and gradient of call(x, ...) against the definition.

    The others' sum is off by SUM; the loss's slope by its logarithm is `other` (parts below), that of a gradient
    Q_j a_j at most Q_j (2 + |a_j| + |other|), with a_j = pull_j / Q_j, 1 at most forwards.  A share w_j is off by
    4 2^-24 of its argument (40 at most) and 2^-23: 1e-5 of itself.
    """
    dtype = logits.dtype
    x = (logits if x is None else x).detach().requires_grad_()
    out = call(x, mask=mask, tau=tau, direction=direction, rest=rest, reduction=reduction)
    want, parts = oracle.distill(array(logits), logp, tokens, mask, tau, direction, rest, reduction)
    other = np.zeros(logits.shape[:2])
    for at, p in parts.items():
        if at != "weight":
            other[at] = abs(p["other"])
    weight = parts["weight"]
    bound = weight * SUM * (1 + other)
    if reduction != "none":
        bound = bound.sum(1)
    got = array(out)
    assert out.dtype == torch.float32 and got.shape == want.shape
    same = got == want  # infinities among them
    with np.errstate(invalid="ignore"):
        assert (same | (np.abs(got - want) <= bound + 2.0**-24 * np.abs(want) + 1e-12)).all(), np.abs(got - want).max()
    rng = np.random.default_rng(seed)
    up = (0.5 + rng.random(want.shape)).astype(np.float32)
    (g,) = torch.autograd.grad([out], [x], [torch.as_tensor(up).to(x.device)])
    assert g.dtype == dtype and g.shape == x.shape
    og = oracle.distill_grad(logits.shape, parts, up, tau)
    half = 2.0**-24 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = 1e-37 if dtype == torch.float32 else float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    tol = (half + 1e-5) * np.abs(og) + tiny
    c = np.abs((up if up.ndim == 2 else up[:, None]) * weight / tau)
    for at, p in parts.items():
        if at == "weight":
            continue
        with np.errstate(invalid="ignore", divide="ignore"):
            a = np.where(p["Q"] > 0, np.abs(p["pull"] / p["Q"]), 0.0) if direction == "reverse" else 1.0
        tol[at] += c[at] * p["Q"] * SUM * (2 + a + abs(p["other"]))
    err = np.abs(array(g) - og)
    assert (err <= tol).all(), (err - tol).max()
    assert (array(g)[weight == 0] == 0).all()
    return out.detach(), g


def check_beam(r, logits, scores, n, tau=1.0, finished=None, eos=None):
    """Totals to the errors of the sum, of the share and half a step of fp32; the continuation in a place has the
    total of the place."""
    s = np.asarray(scores, np.float32).astype(np.float64)
    want, beams, tokens, done = oracle.beam_step(array(logits), s, n, tau, finished, eos)
    totals = oracle.beam_totals(array(logits), s, tau, finished, eos)
    got, gb, gt = array(r.scores), r.beams.cpu().numpy(), r.tokens.cpu().numpy()
    assert r.scores.dtype == torch.float32 and r.beams.dtype == torch.int32 and r.tokens.dtype == torch.int32
    assert got.shape == want.shape and gb.shape == want.shape and gt.shape == want.shape
    full = beams >= 0
    assert np.array_equal(gb >= 0, full) and np.array_equal(gt >= 0, full) and (got[~full] == -np.inf).all()
    with np.errstate(invalid="ignore"):
        gap = SUM + share_error(array(logits), beams, tokens, tau) + 2.0**-24 * np.abs(want)
    assert (np.abs(got[full] - want[full]) <= gap[full]).all()
    for b, e in zip(*np.nonzero(full)):
        assert abs(totals[b, gb[b, e], gt[b, e]] - want[b, e]) <= 2 * gap[b, e]
    for b in range(len(want)):  # every continuation once
        pairs = [(w, v) for w, v in zip(gb[b], gt[b]) if w >= 0]
        assert len(set(pairs)) == len(pairs)
    if eos is None:
        assert r.finished is None
    else:
        assert r.finished.dtype == torch.bool
        was = np.zeros(gb.shape, bool) if finished is None else np.take_along_axis(np.asarray(finished), np.maximum(gb, 0), 1)
        assert np.array_equal(r.finished.cpu().numpy(), full & ((gt == eos) | was))
    return beams, tokens
