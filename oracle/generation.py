"""TEST INFRASTRUCTURE ONLY — numpy float64 definitions of the top log-probabilities,
the distillation loss with its gradient written out, and the steps of a beam search.

Only ``tests/`` imports this module; the product never does.  The gradient is pinned by
central differences of the loss in tests/test_generation_ops.py.
"""

from __future__ import annotations

import numpy as np


def log_softmax(x):
    """Rows of x; a row of -inf alone is NaN, as are rows that hold NaN or +inf."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = x.max(-1, keepdims=True)
        d = x - np.where(top == -np.inf, 0.0, top)
        return d - np.log(np.exp(d).sum(-1, keepdims=True))


def best(x, k):
    """Indices of the k largest entries of a row, equal ones by the lowest; not -inf, not NaN."""
    can = np.flatnonzero(x > -np.inf)
    return can[np.argsort(-x[can], kind="stable")][:k]


def top_logp(logits, k, tau=1.0, mask=None):
    """logits (B, S, V) -> (logp, tokens) (B, S, k)."""
    x = np.asarray(logits, np.float64)
    B, S, V = x.shape
    logp, tokens = np.full((B, S, k), -np.inf), np.full((B, S, k), -1, np.int64)
    for b in range(B):
        for s in range(S):
            if mask is not None and not mask[b, s]:
                continue
            at = best(x[b, s], k)
            with np.errstate(invalid="ignore"):
                logp[b, s, : len(at)] = log_softmax(x[b, s] / tau)[at]
            tokens[b, s, : len(at)] = at
    return logp, tokens


def distill(logits, logp, tokens, mask=None, tau=1.0, direction="forward", rest="bucket", reduction="mean"):
    """-> (loss, parts): parts of each position that has a loss, (b, s) -> dict, and ``weight`` (B, S).

    A dict holds Q (V,), pull (V,): tau times the gradient, and other: the gradient of the tokens that are not
    named, together.
    """
    x = np.asarray(logits, np.float64) / tau
    t = np.asarray(logp, np.float32).astype(np.float64)
    B, S, V = x.shape
    value, weight, parts = np.zeros((B, S)), np.zeros((B, S)), {}
    for b in range(B):
        for s in range(S):
            if mask is not None and not mask[b, s]:
                continue
            names = {}
            for e, v in enumerate(np.asarray(tokens)[b, s]):
                if 0 <= v < V and t[b, s, e] != -np.inf:
                    names.setdefault(int(v), t[b, s, e])
            if not names:
                continue
            weight[b, s] = 1.0
            at, lp = np.array(list(names)), np.array(list(names.values()))
            lq = log_softmax(x[b, s])
            left = np.ones(V, bool)
            left[at] = False
            o = lq[left]
            with np.errstate(invalid="ignore", divide="ignore"):
                top = o.max(initial=-np.inf)
                lqr = -np.inf if top == -np.inf else top + np.log(np.exp(o - top).sum())
                Q, qr = np.exp(lq), np.exp(lqr)
                share = np.zeros(V)
                if lqr > -np.inf or np.isnan(lqr):
                    share[left] = np.exp(log_softmax(x[b, s][left]))  # o - lqr loses it next to huge logits
                if rest == "none":
                    lp = lp - (lp.max() + np.log(np.exp(lp - lp.max()).sum()))
                    pr = 0.0
                else:
                    pr = max(0.0, 1.0 - np.exp(lp).sum())
                P = np.exp(lp)
                pull = np.zeros(V)
                if direction == "forward":
                    v = np.where(P == 0, 0.0, P * (lp - lq[at])).sum()
                    if lqr == -np.inf and pr <= 2.0**-12:
                        pr = 0.0
                    if pr != 0:
                        v += pr * (np.log(pr) - lqr)
                    total = P.sum() + pr  # the loss has no more than these
                    other = total * qr - pr
                    pull[at] = total * Q[at] - P
                else:
                    lpr = np.log(max(pr, 2.0**-24))
                    v = np.where(Q[at] == 0, 0.0, Q[at] * (lq[at] - lp)).sum()
                    if lqr > -np.inf:
                        v += qr * (lqr - lpr)
                    other = 0.0 if lqr == -np.inf else qr * (lqr - lpr - v)
                    pull[at] = np.where(Q[at] == 0, 0.0, Q[at] * (lq[at] - lp - v))
                pull[left] = share[left] * other
            value[b, s] = v
            parts[b, s] = dict(Q=Q, pull=pull, other=other)
    if reduction == "none":
        return value, dict(parts, weight=weight)
    if reduction == "mean":
        weight = weight / np.maximum(weight.sum(1, keepdims=True), 1)
    with np.errstate(invalid="ignore"):
        return np.where(weight > 0, value * weight, 0.0).sum(1), dict(parts, weight=weight)


def distill_grad(shape, parts, grad, tau=1.0):
    """grad (B,) or (B, S); -> d sum(loss grad) / d logits."""
    g = np.asarray(grad, np.float64)
    out = np.zeros(shape)
    for at, p in parts.items():
        if at == "weight":
            continue
        b, s = at
        out[b, s] = p["pull"] * (g[b, s] if g.ndim == 2 else g[b]) * parts["weight"][b, s] / tau
    return out


def beam_totals(logits, scores, tau=1.0, finished=None, eos=None):
    """(B, W, V) totals of all continuations; -inf where there is none."""
    x = np.asarray(logits, np.float64)
    out = np.full(x.shape, -np.inf)
    for b in range(x.shape[0]):
        for w in range(x.shape[1]):
            score = float(scores[b, w])
            if not score > -np.inf:
                continue
            if finished is not None and finished[b, w]:
                out[b, w, eos] = score
                continue
            with np.errstate(invalid="ignore"):
                total = score + log_softmax(x[b, w] / tau)
            out[b, w] = np.where(total > -np.inf, total, -np.inf)
    return out


def beam_step(logits, scores, n, tau=1.0, finished=None, eos=None):
    """-> (scores, beams, tokens, finished) of (B, n)."""
    x = np.asarray(logits, np.float64)
    totals = beam_totals(x, scores, tau, finished, eos)
    B, W, V = x.shape
    out, beams = np.full((B, n), -np.inf), np.full((B, n), -1, np.int64)
    tokens, done = np.full((B, n), -1, np.int64), np.zeros((B, n), bool)
    for b in range(B):
        # by total, then beam, then logit, then token
        w, v = np.nonzero(totals[b] > -np.inf)
        order = np.lexsort((v, -x[b][w, v], w, -totals[b][w, v]))[:n]
        m = len(order)
        w, v = w[order], v[order]
        out[b, :m], beams[b, :m], tokens[b, :m] = totals[b][w, v], w, v
        for e in range(m):
            done[b, e] = (eos is not None and v[e] == eos) or (finished is not None and finished[b, w[e]])
    return out, beams, tokens, done


def beam_reorder(state, beams, lengths=None, dim=None):
    """A new array; the one that is given stays as it is."""
    old, new = np.asarray(state), np.array(state)
    B, W = np.asarray(beams).shape
    for b in range(B):
        for w in range(W):
            p = int(beams[b][w])
            if not 0 <= p < W:
                continue
            if lengths is None:
                new[b, w] = old[b, p]
            else:
                used = [slice(None)] * (old.ndim - 2)
                used[dim - 2] = slice(0, max(0, int(lengths[b])))
                new[(b, w, *used)] = old[(b, p, *used)]
    return new
