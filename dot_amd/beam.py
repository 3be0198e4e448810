"""Beam search: the best continuations of a step, and the states that follow them.

    scores = torch.full((B, W), -inf); scores[:, 0] = 0      # one hypothesis to begin with
    for s in range(steps):
        logits = model(tokens, cache)                        # (B, W, V)
        r = beam_step(logits, scores, finished=finished, eos=eos)
        beam_reorder([tokens, *cache], r.beams)              # in place
        tokens[:, :, s] = r.tokens
        scores, finished = r.scores, r.finished

The hypotheses are answers for a student to train on, or the two sets of a
:func:`preference_loss` over a plan; ``sequence_logp`` of a hypothesis is its score.
Both calls can be captured into a graph.  No counterpart in the reference.
"""

from dataclasses import dataclass
from typing import Optional, Sequence, Union

import torch

from . import _ops
from .distillation import MAX_TOP, _check_logits, _count

MAX_BEAMS = 128


@dataclass
class BeamResult:
    """Result of :func:`beam_step`, by descending score.

    Attributes:
        scores: (B, k) fp32 totals, -inf in empty slots
        beams: (B, k) int32 beam that is continued, -1 in empty slots
        tokens: (B, k) int32 its next token, -1 in empty slots
        finished: (B, k) bool, or None without ``eos``
    """

    scores: torch.Tensor
    beams: torch.Tensor
    tokens: torch.Tensor
    finished: Optional[torch.Tensor] = None


def beam_step(
    logits: torch.Tensor,
    scores: torch.Tensor,
    *,
    k: Optional[int] = None,
    tau: float = 1.0,
    finished: Optional[torch.Tensor] = None,
    eos: Optional[int] = None,
) -> BeamResult:
    """The ``k`` best of all continuations of a batch element's hypotheses by one token.

    A continuation's total is ``scores[w] + log softmax(logits[w] / tau)[v]``, of logits that
    are scaled in fp32; totals are formed and compared in 64 bits, equal ones ordered by beam,
    then by descending logit, then by token.

    Args:
        logits: (B, W, V) or (W, V) in fp32, fp16 or bf16; rows of unit stride are read in
            place.  At most 128 beams; on a GPU V is at most 2^24 and B W at most 2^23.
        scores: (B, W) or (W,) floating point, computed in fp32.  -inf closes a beam: it has no
            continuation and its logits are not read.
        k: Continuations to return (at most 256), W by default; more than W leave room for the
            finished ones among them
        tau: Temperature (> 0; in [1e-20, 1e20] on a GPU)
        finished: Optional bool, shaped as ``scores``: a hypothesis that is finished goes on as
            it is, with token ``eos`` and the same score; its logits are not read
        eos: Token in [0, V) that finishes a hypothesis

    A logit of -inf or NaN is never taken, and a row with a NaN or +inf among its logits has no
    continuation.  A batch element with fewer than ``k`` has empty slots.  No gradient flows
    through the result.
    """
    tau = _check_logits(logits, tau, "W")
    W, V = logits.shape[-2:]
    if not 1 <= W <= MAX_BEAMS:
        raise ValueError(f"between 1 and {MAX_BEAMS} beams are supported, got {W}")
    if not scores.is_floating_point() or scores.shape != logits.shape[:-1]:
        raise ValueError(f"scores must be floating point of shape {tuple(logits.shape[:-1])}, got {scores.dtype} "
                         f"{tuple(scores.shape)}")
    if k is None:
        k = W
    _count(k, min(W * V, MAX_TOP), "k")
    if eos is not None and (isinstance(eos, bool) or not isinstance(eos, int) or not 0 <= eos < V):
        raise ValueError(f"eos must be an int in [0, {V}), got {eos!r}")
    if finished is not None:
        if finished.dtype != torch.bool or finished.shape != scores.shape:
            raise ValueError(f"finished must be bool of shape {tuple(scores.shape)}, got {finished.dtype} "
                             f"{tuple(finished.shape)}")
        if eos is None:
            raise ValueError("finished needs eos")
    batched = logits.dim() == 3
    logits, scores = logits.detach(), scores.detach()
    if not batched:
        logits, scores = logits.unsqueeze(0), scores.unsqueeze(0)
        finished = None if finished is None else finished.unsqueeze(0)
    out = _ops.fused.beam_step(logits, scores, k, tau, finished, -1 if eos is None else eos)
    return BeamResult(*(out if batched else [t.squeeze(0) for t in out]))


def beam_reorder(
    states: Union[torch.Tensor, Sequence[torch.Tensor]],
    beams: torch.Tensor,
    *,
    lengths: Optional[torch.Tensor] = None,
    dim: Optional[int] = None,
) -> None:
    """Gives every beam the states of the beam that it continues, in place:
    ``state[b, w] = state[b, beams[b, w]]`` for all states at once.

    Args:
        states: A tensor or a list of tensors of shape (B, W, ...), of any types: tokens so far,
            keys and values (split a merged first dimension by ``cache.unflatten(0, (B, W))``).
            They may be views, the beams not innermost and of any strides, as long as the other
            dimensions are a run of neighbouring elements and at most one further dimension
            besides that of the positions.  No two places may share memory; states may lie in
            each other's gaps (keys and values of one tensor, of different widths or heads too).
        beams: int32 or int64 (B, W), such as ``beam_step(...).beams``; at most 128 beams.  A beam
            whose entry is outside [0, W) (an empty slot) stays as it is.
        lengths: Optional int32 or int64 (B,): the positions of each batch element that are in
            use; those behind them stay as they are
        dim: Dimension of the positions in every state; ``lengths`` needs it

    Beams that stay what they are are not written, and positions that are not moved not read.
    States that require a gradient are refused while gradients are recorded.
    """
    states = [states] if isinstance(states, torch.Tensor) else list(states)
    if beams.dtype not in (torch.int32, torch.int64) or beams.dim() != 2:
        raise ValueError(f"beams must be int32 or int64 of shape (B, W), got {beams.dtype} {tuple(beams.shape)}")
    if not 1 <= beams.size(1) <= MAX_BEAMS:
        raise ValueError(f"between 1 and {MAX_BEAMS} beams are supported, got {beams.size(1)}")
    if lengths is not None:
        if dim is None:
            raise ValueError("lengths needs dim")
        if lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != beams.shape[:1]:
            raise ValueError(f"lengths must be int32 or int64 of shape ({beams.size(0)},), got {lengths.dtype} "
                             f"{tuple(lengths.shape)}")
    if dim is not None and (isinstance(dim, bool) or not isinstance(dim, int)):
        raise ValueError(f"dim must be an int, got {dim!r}")
    # the states themselves are looked over by the operator: a step has those of all layers
    if states:
        _ops.fused.beam_reorder(states, beams, lengths, dim)
