"""Preference loss over pairs of answers or over a transport plan between two sets.

    ratio = sequence_logp(logits, tokens, ref_logp=ref, mask=answer)    # (2 P,)
    loss = preference_loss(ratio, beta=0.1)                             # (P,) pairs
    loss.mean().backward()

    # P preferred and Q other answers that are no pairs: coupled by a plan
    gap = ratio[:P, None] - ratio[None, P:]
    plan = sinkhorn(softplus(-0.1 * gap), reg=0.1).transport_plan
    loss = preference_loss(ratio, plan=plan, beta=0.1)

``sequence_logp`` gives log-probabilities of token sequences from logits, less
those of a reference model; ``preference_loss`` the loss on these log ratios.
No counterpart in the reference.
"""

from typing import Optional

import torch
import torch.nn as nn

from . import _ops

_REDUCTION = {"none": 0, "sum": 1, "mean": 2}
_LOSS = {"sigmoid": 0, "hinge": 1, "square": 2}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)

# What a call on a GPU takes at most.
MAX_POSITIONS = 1 << 23
MAX_ANSWERS = 1 << 22
_MIN_BETA, _MAX_BETA = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


def sequence_logp(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    *,
    ref_logp: Optional[torch.Tensor] = None,
    mask: Optional[torch.Tensor] = None,
    tau: float = 1.0,
    reduction: str = "sum",
) -> torch.Tensor:
    """Log-probabilities of token sequences, or their log ratios to a reference model.

    ``log softmax(logits / tau)[token]`` of each position, less ``ref_logp``, summed
    over the positions of each sequence in 64 bits.

    Args:
        logits: (B, S, V) or (S, V) in fp32, fp16 or bf16; position s predicts
            ``tokens[..., s]`` (shift them before the call).  A view such as
            ``logits[:, :-1]`` is read in place (one whose last dimension has a stride is
            copied first).  At most 2^23 positions on a GPU.
        tokens: int32 or int64 (B, S) or (S,)
        ref_logp: Optional log-probabilities to subtract, a constant of the gradient:
            per position, shaped as ``tokens`` (``reduction="none"`` of the reference
            model), or one per sequence, (B,) or 0-dim, in the reduction's own scale.
            A log ratio is the small difference of large sums, so per-position values
            (or fp64 sums) keep digits that an fp32 sum has lost.
        mask: Optional bool, shaped as ``tokens``; positions that are False are left
            out (prompt, padding), and so are those whose token is outside [0, V).
            Their logits are not read and their gradient is 0.
        tau: Temperature (> 0; in [1e-20, 1e20] on a GPU)
        reduction: ``"sum"`` or ``"mean"`` over the positions of a sequence (0 for none),
            or ``"none"`` for each position (0 where left out)

    Returns:
        fp32 (B,), 0-dim for unbatched logits, or shaped as ``tokens`` for ``"none"``
    """
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTION)}, got {reduction!r}")
    if logits.dim() not in (2, 3) or logits.size(-1) < 1:
        raise ValueError(f"logits must have shape (B, S, V) or (S, V) with V >= 1, got {tuple(logits.shape)}")
    if logits.dtype not in _FLOATS:
        raise ValueError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens must be int32 or int64 of shape {tuple(logits.shape[:-1])}, got {tokens.dtype} "
                         f"{tuple(tokens.shape)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != tokens.shape):
        raise ValueError(f"mask must be bool of shape {tuple(tokens.shape)}, got {mask.dtype} {tuple(mask.shape)}")
    tau = float(tau)
    if not 0.0 < tau < float("inf"):
        raise ValueError(f"tau must be > 0, got {tau}")
    if logits.is_cuda:
        if not 1e-20 <= tau <= 1e20:
            raise ValueError(f"tau must be in [1e-20, 1e20] on a GPU, got {tau}")
        if tokens.numel() > MAX_POSITIONS:
            raise ValueError(f"at most {MAX_POSITIONS} positions are supported on a GPU, got {tokens.numel()}")
    batched = logits.dim() == 3
    if ref_logp is not None:
        if not ref_logp.is_floating_point() or ref_logp.shape not in (tokens.shape, tokens.shape[:-1]):
            raise ValueError(f"ref_logp must be floating point of shape {tuple(tokens.shape)} or "
                             f"{tuple(tokens.shape[:-1])}, got {ref_logp.dtype} {tuple(ref_logp.shape)}")
        if reduction == "none" and ref_logp.shape != tokens.shape:
            raise ValueError("reduction='none' needs ref_logp per position")
        ref_logp = ref_logp.detach()
    if not batched:
        logits, tokens = logits.unsqueeze(0), tokens.unsqueeze(0)
        mask = None if mask is None else mask.unsqueeze(0)
        ref_logp = None if ref_logp is None else ref_logp.unsqueeze(0)
    out = _ops.fused.sequence_logp_forward(logits, tokens, ref_logp, mask, tau, _REDUCTION[reduction], False)[0]
    return out if batched else out.squeeze(0)


def preference_loss(
    log_ratio: torch.Tensor,
    *,
    plan: Optional[torch.Tensor] = None,
    beta: float = 0.1,
    loss_type: str = "sigmoid",
    label_smoothing: float = 0.0,
) -> torch.Tensor:
    """Loss of preferring the first answers over the others, from their log ratios.

    With ``d`` the difference of two log ratios, ``f(d)`` is

    * ``"sigmoid"``: ``(1 - s) softplus(-beta d) + s softplus(beta d)``, ``s`` the label smoothing
    * ``"hinge"``: ``max(0, 1 - beta d)``
    * ``"square"``: ``(d - 1 / (2 beta))^2``

    Args:
        log_ratio: (P + Q,) log ratios (:func:`sequence_logp`), first of the P preferred,
            then of the Q other answers; floating point, computed in fp32.  P and Q are at
            most 2^22 on a GPU.
        plan: Optional (P, Q) coupling of the two sets, such as the ``transport_plan``
            of :func:`sinkhorn`; without it answer i is paired with answer P + i (P = Q).
            An entry of 0 leaves its pair out, whatever their ratios (a padded answer
            has a row or a column of 0); its own gradient is ``f`` where that is finite.
        beta: Scale (> 0; a normal fp32 number on a GPU)
        loss_type: ``"sigmoid"``, ``"hinge"`` or ``"square"``
        label_smoothing: In [0, 1), ``"sigmoid"`` only

    Returns:
        fp32 (P,): ``f`` of each pair, or ``sum_j plan[i, j] f(log_ratio[i] - log_ratio[P + j])``.
        Gradients reach ``log_ratio`` and ``plan``.
    """
    if loss_type not in _LOSS:
        raise ValueError(f"loss_type must be one of {sorted(_LOSS)}, got {loss_type!r}")
    if log_ratio.dim() != 1 or not log_ratio.is_floating_point():
        raise ValueError(f"log_ratio must be a floating point vector, got {log_ratio.dtype} {tuple(log_ratio.shape)}")
    if plan is None:
        if log_ratio.size(0) % 2:
            raise ValueError(f"pairs need an even number of log ratios, got {log_ratio.size(0)}")
    elif plan.dim() != 2 or not plan.is_floating_point() or sum(plan.shape) != log_ratio.size(0):
        raise ValueError(f"plan must be floating point of shape (P, Q) with P + Q = {log_ratio.size(0)}, got "
                         f"{plan.dtype} {tuple(plan.shape)}")
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not 0.0 < beta < float("inf"):
        raise ValueError(f"beta must be > 0, got {beta}")
    if log_ratio.is_cuda:
        if not _MIN_BETA <= beta <= _MAX_BETA:
            raise ValueError(f"beta must be a normal fp32 number on a GPU, got {beta}")
        if log_ratio.size(0) > MAX_ANSWERS:
            answers = max(plan.shape) if plan is not None else log_ratio.size(0) // 2
            if answers > MAX_ANSWERS:
                raise ValueError(f"at most {MAX_ANSWERS} answers of a set are supported on a GPU, got {answers}")
    if not 0.0 <= label_smoothing < 1.0:
        raise ValueError(f"label_smoothing must be in [0, 1), got {label_smoothing}")
    if label_smoothing and loss_type != "sigmoid":
        raise ValueError("label_smoothing needs loss_type='sigmoid'")
    return _ops.fused.preference_forward(log_ratio, plan, _LOSS[loss_type], beta, label_smoothing)


class SequenceLogp(nn.Module):
    """Module wrapper of :func:`sequence_logp`."""

    def __init__(self, tau: float = 1.0, reduction: str = "sum"):
        super().__init__()
        self.tau = tau
        self.reduction = reduction

    def forward(self, logits: torch.Tensor, tokens: torch.Tensor, ref_logp: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        return sequence_logp(logits, tokens, ref_logp=ref_logp, mask=mask, tau=self.tau, reduction=self.reduction)


class PreferenceLoss(nn.Module):
    """Module wrapper of :func:`preference_loss`."""

    def __init__(self, beta: float = 0.1, loss_type: str = "sigmoid", label_smoothing: float = 0.0):
        super().__init__()
        self.beta = beta
        self.loss_type = loss_type
        self.label_smoothing = label_smoothing

    def forward(self, log_ratio: torch.Tensor, plan: Optional[torch.Tensor] = None) -> torch.Tensor:
        return preference_loss(log_ratio, plan=plan, beta=self.beta, loss_type=self.loss_type,
                               label_smoothing=self.label_smoothing)
