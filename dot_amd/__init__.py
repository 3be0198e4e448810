"""dot_amd — differentiable optimal transport on AMD MI355X (gfx950).

A from-scratch MI355X implementation of DOT's batched Sinkhorn and
bidirectional-softmax operators with the reference's Python API:

    result = dot_amd.sinkhorn(cost, reg=1.0, n_iters=100)   # also max_iter=
    result.transport_plan   # (B, M, N)
    result.cost             # (B,)
    P = dot_amd.bidirectional_softmax(sim, tau=1.0)

and the operators that language models put around a transport plan: routing of
tokens to experts with its balance loss, log-probabilities of sequences and the
preference loss over pairs or over a plan:

    r = dot_amd.topk_routing(scores, k=2)        # weights, experts, counts, balance_loss
    ratio = dot_amd.sequence_logp(logits, tokens, ref_logp=ref)
    loss = dot_amd.preference_loss(ratio, plan=plan)

and what makes and teaches the answers: distillation from a teacher's top
log-probabilities, and the steps of a beam search:

    teacher = dot_amd.top_logp(teacher_logits, k=64)      # logp, tokens
    loss = dot_amd.distill_loss(logits, teacher.logp, teacher.tokens)
    r = dot_amd.beam_step(logits, scores)                 # scores, beams, tokens
    dot_amd.beam_reorder([tokens, *cache], r.beams)       # in place

The operators are registered as ``torch.ops.dot.*`` (the reference's schemas)
and run hand-written HIP kernels behind the C ABI in ``include/dot_amd.h``.
``import dot`` gives the same API under the reference's package name.
"""

# Load the operator library first (raises ImportError when it is not built).
from . import _ops

from .sinkhorn import (
    sinkhorn,
    sinkhorn_from_scores,
    spectral_preflight,
    SinkhornResult,
    Sinkhorn,
    SinkhornFromScores,
)
from .bidirectional_softmax import (
    bidirectional_softmax,
    bidirectional_softmax_with_lengths,
    BidirectionalSoftmax,
)
from .routing import (
    topk_routing,
    balance_loss,
    RoutingResult,
    BalanceResult,
    TopKRouting,
    BalanceLoss,
)
from .preference import (
    sequence_logp,
    preference_loss,
    SequenceLogp,
    PreferenceLoss,
)
from .distillation import (
    top_logp,
    distill_loss,
    TopLogpResult,
    TopLogp,
    DistillLoss,
)
from .beam import (
    beam_step,
    beam_reorder,
    BeamResult,
)

__version__ = "0.1.0"

__all__ = [
    "sinkhorn",
    "sinkhorn_from_scores",
    "spectral_preflight",
    "SinkhornResult",
    "Sinkhorn",
    "SinkhornFromScores",
    "bidirectional_softmax",
    "bidirectional_softmax_with_lengths",
    "BidirectionalSoftmax",
    "topk_routing",
    "balance_loss",
    "RoutingResult",
    "BalanceResult",
    "TopKRouting",
    "BalanceLoss",
    "sequence_logp",
    "preference_loss",
    "SequenceLogp",
    "PreferenceLoss",
    "top_logp",
    "distill_loss",
    "TopLogpResult",
    "TopLogp",
    "DistillLoss",
    "beam_step",
    "beam_reorder",
    "BeamResult",
]
