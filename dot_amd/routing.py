"""Routing of tokens to experts: top-k selection, its weights and the balance loss.

    r = topk_routing(scores, k=2)             # router logits (B, N, E)
    r.weights, r.experts                      # (B, N, k)
    r.counts, r.balance_loss                  # (B, E), (B,)

    plan = sinkhorn_from_scores(logits, tau=0.5)
    r = topk_routing(plan, k=2, scoring="plan", normalize=True)

The scores of a token are router logits or its row of a transport plan (what
``sinkhorn_from_scores`` gives for balanced routing).  With the mass
``q = softmax(s)``, ``sigmoid(s)`` or ``s`` itself, the share ``p = q / sum q``
and ``n`` unmasked tokens, the balance loss of a batch element is

    E * sum_e (counts_e / (k n)) * (sum_i p_ie / n)

which is 1 for a balanced assignment.  Counts are constants of its gradient.
No counterpart in the reference.
"""

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn

from . import _ops

MAX_EXPERTS = 4096
MAX_K = 64

_SCORING = {"softmax": 0, "sigmoid": 1, "plan": 2}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


@dataclass
class RoutingResult:
    """Result of :func:`topk_routing`; without a batch dimension for 2D scores.

    Attributes:
        weights: (B, N, k) fp32 masses of the selected experts, 0 in empty slots
        experts: (B, N, k) int32 selected experts by descending key, -1 in empty slots
        counts: (B, E) int32 slots that each expert got
        balance_loss: (B,) fp32
    """

    weights: torch.Tensor
    experts: torch.Tensor
    counts: torch.Tensor
    balance_loss: torch.Tensor


@dataclass
class BalanceResult:
    """Result of :func:`balance_loss`: ``loss`` (B,) fp32 and ``counts`` (B, E) int32."""

    loss: torch.Tensor
    counts: torch.Tensor


def _check_scores(scores, scoring, mask):
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {sorted(_SCORING)}, got {scoring!r}")
    if scores.dim() not in (2, 3):
        raise ValueError(f"scores must have shape (B, N, E) or (N, E), got {tuple(scores.shape)}")
    if scores.dtype not in _FLOATS:
        raise ValueError(f"scores must be float32, float16 or bfloat16, got {scores.dtype}")
    if not 1 <= scores.size(-1) <= MAX_EXPERTS:
        raise ValueError(f"between 1 and {MAX_EXPERTS} experts are supported, got {scores.size(-1)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != scores.shape[:-1]):
        raise ValueError(f"mask must be bool of shape {tuple(scores.shape[:-1])}, got {mask.dtype} "
                         f"{tuple(mask.shape)}")


def topk_routing(
    scores: torch.Tensor,
    k: int,
    *,
    scoring: str = "softmax",
    normalize: bool = False,
    bias: Optional[torch.Tensor] = None,
    mask: Optional[torch.Tensor] = None,
) -> RoutingResult:
    """The ``k`` experts of each token, their weights, per-expert counts and the balance loss.

    Args:
        scores: (B, N, E) or (N, E) in fp32, fp16 or bf16; the last dimension of any
            stride, at most 4096 experts
        k: Experts per token (at most 64)
        scoring: Mass of a score: ``"softmax"`` over the row, ``"sigmoid"``, or
            ``"plan"`` for rows of a transport plan (masses as they are)
        normalize: Weights of a token sum to 1
        bias: Optional (E,) added to the scores themselves, whatever the scoring, for the
            selection only (a column potential, -inf to close an expert); it gets no
            gradient.  Routers that are balanced by a bias on the masses,
            ``sigmoid(logit) + bias``, select by another order: form the masses first,
            ``topk_routing(torch.sigmoid(logits.float()), k, scoring="plan", bias=bias)``,
            which selects by ``mass + bias`` and has the same weights, loss and gradient
        mask: Optional bool (B, N); tokens that are False are left out: experts -1,
            weights 0, not counted, gradient 0.  Their scores are not read.

    Experts are ordered by ``score + bias`` in fp32, equal ones by the lowest index.
    One is available where that is above -inf (and, with ``"plan"``, its mass above
    0); a token with fewer than ``k`` has empty slots.  Masses that sum to less than
    the smallest normal fp32 (1.2e-38) count as none, a token's own as well as those
    of its experts that ``normalize`` divides by: their weights and shares are 0, and so
    is the gradient through them.  A sigmoid mass below that is 0.  A NaN score is never
    selected; its token's softmax weights and the loss are NaN.

    Gradients reach ``scores`` from ``weights`` and ``balance_loss``.
    """
    _check_scores(scores, scoring, mask)
    if isinstance(k, bool) or not isinstance(k, int) or not 1 <= k <= min(scores.size(-1), MAX_K):
        raise ValueError(f"k must be an int in [1, {min(scores.size(-1), MAX_K)}], got {k!r}")
    if bias is not None:
        if bias.shape != scores.shape[-1:] or not bias.is_floating_point():
            raise ValueError(f"bias must be floating point of shape ({scores.size(-1)},), got {tuple(bias.shape)}")
        bias = bias.detach()
    batched = scores.dim() == 3
    if not batched:
        scores, mask = scores.unsqueeze(0), None if mask is None else mask.unsqueeze(0)
    counts, loss, weights, experts = _ops.fused.routing_forward(scores, k, _SCORING[scoring], normalize, bias, mask,
                                                                None)[:4]
    if not batched:
        weights, experts, counts, loss = (x.squeeze(0) for x in (weights, experts, counts, loss))
    return RoutingResult(weights, experts, counts, loss)


def balance_loss(
    scores: torch.Tensor,
    experts: torch.Tensor,
    *,
    scoring: str = "softmax",
    mask: Optional[torch.Tensor] = None,
) -> BalanceResult:
    """Per-expert counts and the balance loss of a given assignment.

    Args:
        scores: As in :func:`topk_routing`
        experts: int32 or int64 (B, N, k) or (N, k); entries outside [0, E) (such as
            the -1 of an empty slot) are not counted, one that a token names twice
            counts twice
        scoring, mask: As in :func:`topk_routing`

    The assignment may come from elsewhere than ``scores``: from a transport plan
    of them, from a group-limited choice, from another router.  Gradients reach
    ``scores``.
    """
    _check_scores(scores, scoring, mask)
    if experts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"experts must be int32 or int64, got {experts.dtype}")
    if experts.dim() != scores.dim() or experts.shape[:-1] != scores.shape[:-1]:
        raise ValueError(f"experts must have shape {tuple(scores.shape[:-1])} + (k,), got {tuple(experts.shape)}")
    if not 1 <= experts.size(-1) <= MAX_K:
        raise ValueError(f"between 1 and {MAX_K} experts per token are supported, got {experts.size(-1)}")
    batched = scores.dim() == 3
    if not batched:
        scores, experts = scores.unsqueeze(0), experts.unsqueeze(0)
        mask = None if mask is None else mask.unsqueeze(0)
    counts, loss = _ops.fused.routing_forward(scores, experts.size(-1), _SCORING[scoring], False, None, mask,
                                              experts)[:2]
    return BalanceResult(loss, counts) if batched else BalanceResult(loss.squeeze(0), counts.squeeze(0))


class TopKRouting(nn.Module):
    """Module wrapper of :func:`topk_routing`."""

    def __init__(self, k: int, scoring: str = "softmax", normalize: bool = False):
        super().__init__()
        self.k = k
        self.scoring = scoring
        self.normalize = normalize

    def forward(self, scores: torch.Tensor, bias: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None) -> RoutingResult:
        return topk_routing(scores, self.k, scoring=self.scoring, normalize=self.normalize, bias=bias, mask=mask)


class BalanceLoss(nn.Module):
    """Module wrapper of :func:`balance_loss`."""

    def __init__(self, scoring: str = "softmax"):
        super().__init__()
        self.scoring = scoring

    def forward(self, scores: torch.Tensor, experts: torch.Tensor,
                mask: Optional[torch.Tensor] = None) -> BalanceResult:
        return balance_loss(scores, experts, scoring=self.scoring, mask=mask)
