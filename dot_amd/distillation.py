"""Distillation from a teacher's top log-probabilities.

    with torch.no_grad():
        teacher = top_logp(teacher_logits, k=64)          # logp, tokens: (B, S, 64)
    loss = distill_loss(logits, teacher.logp, teacher.tokens, mask=answer).mean()
    loss.backward()

``top_logp`` gives the k likeliest tokens of each position with their
log-probabilities (a teacher's targets to keep, or what to show beside an answer);
``distill_loss`` the divergence of a student's logits from them, which needs no
second vocabulary of logits in memory.  No counterpart in the reference.
"""

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn as nn

from . import _ops
from .preference import _FLOATS, _REDUCTION, MAX_POSITIONS

MAX_TOP = 256
MAX_VOCABULARY = 1 << 24

_DIRECTION = {"forward": 0, "reverse": 1}
_REST = {"bucket": 0, "none": 1}


@dataclass
class TopLogpResult:
    """Result of :func:`top_logp`, by descending probability.

    Attributes:
        logp: (B, S, k) fp32 log-probabilities, -inf in empty slots
        tokens: (B, S, k) int32, -1 in empty slots
    """

    logp: torch.Tensor
    tokens: torch.Tensor


def _check_logits(logits, tau, last):
    """Checks that logits of (B, S, V) or (S, V), or of beams, have in common."""
    if logits.dim() not in (2, 3) or logits.size(-1) < 1:
        raise ValueError(f"logits must have shape (B, {last}, V) or ({last}, V) with V >= 1, got {tuple(logits.shape)}")
    if logits.dtype not in _FLOATS:
        raise ValueError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    tau = float(tau)
    if not 0.0 < tau < float("inf"):
        raise ValueError(f"tau must be > 0, got {tau}")
    if logits.is_cuda:
        if not 1e-20 <= tau <= 1e20:
            raise ValueError(f"tau must be in [1e-20, 1e20] on a GPU, got {tau}")
        V = logits.size(-1)
        if V > MAX_VOCABULARY:
            raise ValueError(f"at most {MAX_VOCABULARY} tokens of a vocabulary are supported on a GPU, got {V}")
        # rows of more than 2^18 tokens count once for each 2^18
        if logits.shape[:-1].numel() * -(-V // (1 << 18)) > MAX_POSITIONS:
            raise ValueError(f"at most {MAX_POSITIONS} positions are supported on a GPU, got {tuple(logits.shape[:-1])}")
    return tau


def _check_mask(mask, shape):
    if mask is not None and (mask.dtype != torch.bool or mask.shape != shape):
        raise ValueError(f"mask must be bool of shape {tuple(shape)}, got {mask.dtype} {tuple(mask.shape)}")


def _count(n, most, name):
    if isinstance(n, bool) or not isinstance(n, int) or not 1 <= n <= most:
        raise ValueError(f"{name} must be an int in [1, {most}], got {n!r}")


def top_logp(
    logits: torch.Tensor,
    k: int,
    *,
    tau: float = 1.0,
    mask: Optional[torch.Tensor] = None,
) -> TopLogpResult:
    """The ``k`` likeliest tokens of each position and ``log softmax(logits / tau)`` of them.

    Args:
        logits: (B, S, V) or (S, V) in fp32, fp16 or bf16; a view such as ``logits[:, :-1]``
            is read in place (one whose last dimension has a stride is copied first).  On a
            GPU V is at most 2^24, and there are at most 2^23 positions.
        k: Tokens per position (at most 256)
        tau: Temperature (> 0; in [1e-20, 1e20] on a GPU)
        mask: Optional bool (B, S); positions that are False are left out: their slots are
            empty and their logits are not read

    Tokens are ordered by logit, equal ones by the lowest token.  A logit of -inf or NaN is
    never taken; a position with fewer than ``k`` others has empty slots.  The
    log-probabilities of a position that has a NaN or +inf are NaN.  No gradient flows
    through the result.
    """
    tau = _check_logits(logits, tau, "S")
    _check_mask(mask, logits.shape[:-1])
    _count(k, min(logits.size(-1), MAX_TOP), "k")
    batched = logits.dim() == 3
    x = logits.detach()
    if not batched:
        x, mask = x.unsqueeze(0), None if mask is None else mask.unsqueeze(0)
    logp, tokens = _ops.fused.top_logp(x, k, tau, mask)
    return TopLogpResult(logp, tokens) if batched else TopLogpResult(logp.squeeze(0), tokens.squeeze(0))


def distill_loss(
    logits: torch.Tensor,
    teacher_logp: torch.Tensor,
    teacher_tokens: torch.Tensor,
    *,
    mask: Optional[torch.Tensor] = None,
    tau: float = 1.0,
    direction: str = "forward",
    rest: str = "bucket",
    reduction: str = "mean",
) -> torch.Tensor:
    """Divergence of ``softmax(logits / tau)`` from a teacher's top log-probabilities.

    With the teacher's probabilities ``P`` of its K tokens, what they leave
    ``P_r = 1 - sum P`` (0 if rounding makes it less), the student's ``Q`` and its rest
    ``Q_r`` over the tokens that are not the teacher's, a position's divergence is

    * ``"forward"``: ``sum P (log P - log Q) + P_r (log P_r - log Q_r)``
    * ``"reverse"``: ``sum Q (log Q - log P) + Q_r (log Q_r - log P_r)``, with a ``P_r`` of at
      least 2^-24 (what fp32 log-probabilities can tell from nothing)

    Args:
        logits: (B, S, V) or (S, V) in fp32, fp16 or bf16, as in :func:`sequence_logp`.  On a
            GPU V is at most 2^24, and there are at most 2^23 positions.
        teacher_logp: (B, S, K) or (S, K) floating point log-probabilities at the same
            temperature (``top_logp(..., tau=tau).logp``), computed in fp32; constants of the
            gradient.  K is at most 256.  Ones kept in 16 bits are taken as they are, and what
            their rounding leaves of 1 is rest (up to 2^-11 of the list's entropy in fp16, 2^-8
            in bf16): where the list is all that the student allows, use ``rest="none"``.
        teacher_tokens: int32 or int64, shaped as ``teacher_logp``.  An entry whose token is
            outside [0, V) or whose log-probability is -inf names no token, nor does one whose
            token an earlier entry names.
        mask: Optional bool (B, S); positions that are False are left out, and so are those
            that name no token.  Their logits are not read and their gradient is 0.
        tau: Temperature (> 0; in [1e-20, 1e20] on a GPU).  The loss is not multiplied by its
            square.
        direction: ``"forward"`` (mean-seeking) or ``"reverse"`` (mode-seeking)
        rest: ``"bucket"`` for the rest as a class of its own, as above; ``"none"`` makes the
            teacher's K probabilities sum to 1 instead (``"forward"`` only)
        reduction: ``"mean"`` or ``"sum"`` over the positions of a sequence (0 for none), in 64
            bits, or ``"none"`` for each position (0 where left out)

    Returns:
        fp32 (B,), 0-dim for unbatched logits, or (B, S) for ``"none"``.  Where the student
        has no probability for what the teacher has, the divergence is +inf; its gradient
        stays finite.  A rest of the teacher of at most 2^-12 is not held against a student
        that has none: the log-probabilities of :func:`top_logp` leave as much by their
        rounding, 2^-23 times the largest scaled logit.
    """
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTION)}, got {reduction!r}")
    if direction not in _DIRECTION:
        raise ValueError(f"direction must be one of {sorted(_DIRECTION)}, got {direction!r}")
    if rest not in _REST:
        raise ValueError(f"rest must be one of {sorted(_REST)}, got {rest!r}")
    if direction == "reverse" and rest != "bucket":
        raise ValueError("direction='reverse' needs rest='bucket'")
    tau = _check_logits(logits, tau, "S")
    _check_mask(mask, logits.shape[:-1])
    if teacher_tokens.dtype not in (torch.int32, torch.int64) or teacher_tokens.shape[:-1] != logits.shape[:-1]:
        raise ValueError(f"teacher_tokens must be int32 or int64 of shape {tuple(logits.shape[:-1])} + (K,), got "
                         f"{teacher_tokens.dtype} {tuple(teacher_tokens.shape)}")
    if not 1 <= teacher_tokens.size(-1) <= MAX_TOP:
        raise ValueError(f"between 1 and {MAX_TOP} tokens of a position are supported, got {teacher_tokens.size(-1)}")
    if not teacher_logp.is_floating_point() or teacher_logp.shape != teacher_tokens.shape:
        raise ValueError(f"teacher_logp must be floating point of shape {tuple(teacher_tokens.shape)}, got "
                         f"{teacher_logp.dtype} {tuple(teacher_logp.shape)}")
    teacher_logp = teacher_logp.detach()
    batched = logits.dim() == 3
    if not batched:
        logits, teacher_logp, teacher_tokens = logits.unsqueeze(0), teacher_logp.unsqueeze(0), teacher_tokens.unsqueeze(0)
        mask = None if mask is None else mask.unsqueeze(0)
    out = _ops.fused.distill_forward(logits, teacher_logp, teacher_tokens, mask, tau, _DIRECTION[direction],
                                     _REST[rest], _REDUCTION[reduction], False)[0]
    return out if batched else out.squeeze(0)


class TopLogp(nn.Module):
    """Module wrapper of :func:`top_logp`."""

    def __init__(self, k: int, tau: float = 1.0):
        super().__init__()
        self.k = k
        self.tau = tau

    def forward(self, logits: torch.Tensor, mask: Optional[torch.Tensor] = None) -> TopLogpResult:
        return top_logp(logits, self.k, tau=self.tau, mask=mask)


class DistillLoss(nn.Module):
    """Module wrapper of :func:`distill_loss`."""

    def __init__(self, tau: float = 1.0, direction: str = "forward", rest: str = "bucket", reduction: str = "mean"):
        super().__init__()
        self.tau = tau
        self.direction = direction
        self.rest = rest
        self.reduction = reduction

    def forward(self, logits: torch.Tensor, teacher_logp: torch.Tensor, teacher_tokens: torch.Tensor,
                mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        return distill_loss(logits, teacher_logp, teacher_tokens, mask=mask, tau=self.tau, direction=self.direction,
                            rest=self.rest, reduction=self.reduction)
