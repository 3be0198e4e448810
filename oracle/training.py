"""TEST INFRASTRUCTURE ONLY — numpy float64 definitions of the routing, sequence
log-probability and preference operators, with their gradients written out.

Only ``tests/`` imports this module; the product never does.  The gradients are
pinned by central differences of the forwards in tests/test_training_ops.py.
"""

from __future__ import annotations

import numpy as np


def _exp(x):
    with np.errstate(over="ignore", under="ignore", invalid="ignore"):
        return np.exp(x)


def _masses(s, scoring):
    """(q, sum q, dq/ds) of rows of scores; softmax rows of -inf alone have no mass."""
    if scoring == "softmax":
        top = s.max(-1, keepdims=True, initial=-np.inf)
        with np.errstate(invalid="ignore"):
            e = _exp(s - np.where(top == -np.inf, 0.0, top))
        z = e.sum(-1, keepdims=True)
        q = np.where(z == 0, 0.0, e / np.where(z == 0, 1.0, z))
        return q, q.sum(-1, keepdims=True), None
    if scoring == "sigmoid":
        t = _exp(-np.abs(s))
        t = np.where(t < np.finfo(np.float32).tiny, 0.0, t)  # counts as none, as such sums do
        q = np.where(s < 0, t, 1.0) / (1 + t)
        return q, q.sum(-1, keepdims=True), t / (1 + t) ** 2
    q = np.where(s == -np.inf, 0.0, s)
    return q, q.sum(-1, keepdims=True), np.ones_like(s)


def _none(mass):
    """Whether masses sum to less than the smallest normal fp32, and so count as none."""
    return abs(mass) < np.finfo(np.float32).tiny


def route(scores, k, scoring="softmax", normalize=False, bias=None, mask=None, given=None):
    """scores (B, N, E) as float32 values; -> dict of weights, experts, counts, tokens, loss."""
    s32 = np.asarray(scores, dtype=np.float32)
    B, N, E = s32.shape
    s = s32.astype(np.float64)
    live = np.ones((B, N), bool) if mask is None else np.asarray(mask, bool)
    out = dict(counts=np.zeros((B, E), np.int64), tokens=live.sum(1), loss=np.zeros(B))
    if given is None:
        out["weights"] = np.zeros((B, N, k))
        out["experts"] = np.full((B, N, k), -1, np.int64)
        with np.errstate(invalid="ignore", over="ignore"):
            key = s32 + (np.float32(0) if bias is None else np.asarray(bias, np.float32))
    for b in range(B):
        share = np.zeros(E)
        for n in np.flatnonzero(live[b]):
            q, total, _ = _masses(s[b, n], scoring)
            if given is None:
                t = key[b, n]
                can = [e for e in range(E) if t[e] > -np.inf and (scoring != "plan" or s[b, n, e] > 0)]
                took = sorted(can, key=lambda e: (-t[e], e))[:k]
                if took:
                    if normalize and scoring == "softmax":
                        w = _exp(s[b, n, took] - s[b, n, took].max()) + (total - total)
                    else:
                        w = q[took]
                    if normalize:
                        w = 0.0 * w if _none(w.sum()) else w / w.sum()
                    out["weights"][b, n, :len(took)] = w
                    out["experts"][b, n, :len(took)] = took
            else:
                took = [e for e in given[b, n] if 0 <= e < E]
            np.add.at(out["counts"][b], np.asarray(took, dtype=np.int64), 1)
            if not _none(total[0]):
                share += q / total
        n_b = out["tokens"][b]
        if n_b:
            out["loss"][b] = E * (out["counts"][b] / (k * n_b) * (share / n_b)).sum()
    return out


def route_grad(scores, k, fwd, scoring="softmax", normalize=False, mask=None, grad_weights=None, grad_loss=None):
    """d(sum weights grad_weights + sum loss grad_loss) / d scores."""
    s = np.asarray(scores, dtype=np.float64)
    B, N, E = s.shape
    live = np.ones((B, N), bool) if mask is None else np.asarray(mask, bool)
    out = np.zeros_like(s)
    for b in range(B):
        n_b = fwd["tokens"][b]
        h0 = np.zeros(E)
        if grad_loss is not None and n_b:
            h0 = grad_loss[b] * E * fwd["counts"][b] / (k * n_b * n_b)
        for n in np.flatnonzero(live[b]):
            q, total, slope = _masses(s[b, n], scoring)
            h, add = h0.copy(), np.zeros(E)
            if grad_weights is not None:
                at = fwd["experts"][b, n]
                ok = at >= 0
                w, dw, at = fwd["weights"][b, n][ok], grad_weights[b, n][ok], at[ok]
                if normalize:
                    dw = dw - (w * dw).sum()
                    mass = q[at].sum()
                    add[at] = w * dw if scoring == "softmax" else 0.0 if _none(mass) else dw / mass
                elif scoring == "softmax":
                    h[at] += dw
                else:
                    add[at] = dw
            p = 0.0 * q if _none(total[0]) else q / total
            if scoring == "softmax":
                out[b, n] = p * (h - (p * h).sum()) + add
            else:
                back = 0.0 if _none(total[0]) else (h - (p * h).sum()) / total
                out[b, n] = slope * (back + add)
    return out


def sequence_logp(logits, tokens, ref=None, mask=None, tau=1.0, reduction="sum"):
    """-> (out, softmax rows (B, S, V), weight of each position (B, S))."""
    x = np.asarray(logits, dtype=np.float64) / tau
    B, S, V = x.shape
    tokens = np.asarray(tokens)
    live = (tokens >= 0) & (tokens < V)
    if mask is not None:
        live &= np.asarray(mask, bool)
    value, p = np.zeros((B, S)), np.zeros((B, S, V))
    for b, s in zip(*np.nonzero(live)):
        row = x[b, s]
        top = row.max()
        with np.errstate(invalid="ignore"):
            e = _exp(row - (0.0 if top == -np.inf else top))
        p[b, s] = e / e.sum()
        value[b, s] = row[tokens[b, s]] - (0.0 if top == -np.inf else top) - np.log(e.sum())
        if ref is not None and np.ndim(ref) == 2:
            value[b, s] -= float(ref[b, s])
    weight = live.astype(np.float64)
    if reduction == "none":
        return value, p, weight
    if reduction == "mean":
        weight = weight / np.maximum(live.sum(1, keepdims=True), 1)
    out = (value * weight).sum(1)
    if ref is not None and np.ndim(ref) == 1:
        out = out - np.asarray(ref, np.float64)
    return out, p, weight


def sequence_logp_grad(p, weight, tokens, grad, tau=1.0):
    """grad (B,) or (B, S); -> d sum(out grad) / d logits."""
    g = np.asarray(grad, np.float64)
    c = (g if g.ndim == 2 else g[:, None]) * weight / tau
    out = -p * c[:, :, None]
    for b, s in zip(*np.nonzero(weight)):
        out[b, s, tokens[b, s]] += c[b, s]
    out[weight == 0] = 0.0
    return out


def preference(ratio, plan=None, beta=0.1, loss_type="sigmoid", smoothing=0.0, grad=None):
    """-> (loss (P,), grad_ratio, grad_plan); gradients of sum(loss grad)."""
    r = np.asarray(ratio, np.float64)
    P = len(r) // 2 if plan is None else len(plan)
    with np.errstate(invalid="ignore"):
        gap = r[:P] - r[P:] if plan is None else r[:P, None] - r[None, P:]
    d = beta * gap
    if loss_type == "sigmoid":
        t = _exp(-np.abs(d))
        up = np.where(d < 0, t, 1.0) / (1 + t)
        down = np.where(d < 0, 1.0, t) / (1 + t)
        f = np.log1p(t) + (1 - smoothing) * np.maximum(-d, 0)
        if smoothing:
            f = f + smoothing * np.maximum(d, 0)
        slope = beta * (smoothing * up - (1 - smoothing) * down)
    elif loss_type == "hinge":
        f = np.maximum(0, 1 - d)
        slope = np.where(d < 1, -beta, 0.0)
    else:
        f = (gap - 0.5 / beta) ** 2
        slope = 2 * (gap - 0.5 / beta)
    g = np.ones(P) if grad is None else np.asarray(grad, np.float64)
    if plan is None:
        return f, np.concatenate([g * slope, -g * slope]), None
    plan = np.asarray(plan, np.float64)
    out = plan == 0  # leaves the pair out
    pull = plan * np.where(out, 0.0, slope) * g[:, None]
    own = np.where(out & ~(f < np.inf), 0.0, f) * g[:, None]
    return (plan * np.where(out, 0.0, f)).sum(1), np.concatenate([pull.sum(1), -pull.sum(0)]), own
