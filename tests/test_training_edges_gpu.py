"""The routing, sequence log-probability and preference operators on the device where
their rules decide, against the float64 definition."""

import numpy as np
import pytest
import torch

import dot_amd
from conftest import rel_err
from oracle import training as oracle
from test_training_edges import small_rows

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("scoring", ["plan", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
def test_masses_below_the_smallest_normal_count_as_none(scoring, normalize):
    """As on the CPU.  Sums and products of 8 terms and an exponential to (|d| + 8) 2^-24 of itself, 6e-6 at -87: 1e-5."""
    s = small_rows(scoring)
    x = torch.as_tensor(s).to(DEV).requires_grad_()
    r = dot_amd.topk_routing(x, 2, scoring=scoring, normalize=normalize)
    o = oracle.route(s, 2, scoring, normalize)
    assert np.array_equal(r.experts.cpu().numpy(), o["experts"])
    assert rel_err(r.weights, o["weights"]) < 1e-5 and rel_err(r.balance_loss, o["loss"]) < 1e-5
    none = [1, 3, 4]
    if normalize:
        assert (r.weights[0, none] == 0).all()
        assert rel_err(r.weights[0, [0, 2, 5]].sum(-1), torch.ones(3)) < 1e-5
    rng = np.random.default_rng(1)
    dw, dl = rng.standard_normal(o["weights"].shape).astype(np.float32), np.ones(1, np.float32)
    (g,) = torch.autograd.grad([r.weights, r.balance_loss], [x],
                               [torch.as_tensor(dw).to(DEV), torch.as_tensor(dl).to(DEV)])
    og = oracle.route_grad(s, 2, o, scoring, normalize, None, dw, dl)
    assert torch.isfinite(g).all()
    assert rel_err(g[0, [0, 5]], og[0, [0, 5]]) < 1e-5 and rel_err(g[0, 2], og[0, 2]) < 1e-5
    err = np.abs(g[0, none].cpu().double().numpy() - og[0, none])
    assert (err <= 1e-5 * np.abs(og[0, none]).max() + 2.0**-126).all()
    if normalize:
        assert (g[0, none] == 0).all()
    q = dot_amd.balance_loss(x[:, none], torch.zeros(1, 3, 1, dtype=torch.int32, device=DEV), scoring=scoring)
    assert q.loss.tolist() == [0.0] and q.counts[0].tolist() == [3] + [0] * 7
    assert (torch.autograd.grad(q.loss.sum(), x)[0] == 0).all()


def test_limits_of_the_device_are_refused_as_values():
    """Before any launch, as other arguments are; on the CPU the same calls run."""
    x, tokens = torch.zeros(1, 2, 4), torch.zeros(1, 2, dtype=torch.long)
    for tau in (1e-21, 1e21):
        assert torch.isfinite(dot_amd.sequence_logp(x, tokens, tau=tau)).all()
        with pytest.raises(ValueError, match="tau"):
            dot_amd.sequence_logp(x.to(DEV), tokens.to(DEV), tau=tau)
    for tau in (1e-20, 1e20):
        assert torch.isfinite(dot_amd.sequence_logp(x.to(DEV), tokens.to(DEV), tau=tau)).all()
    few = torch.zeros(1, 1, 1, device=DEV).expand(1, 2**23 + 1, 1)
    with pytest.raises(ValueError, match="positions"):
        dot_amd.sequence_logp(few, torch.zeros(1, 1, dtype=torch.int32, device=DEV).expand(1, 2**23 + 1))
    ratio = torch.zeros(4)
    for beta in (1e-39, 1e39):
        assert dot_amd.preference_loss(ratio, beta=beta).shape == (2,)
        with pytest.raises(ValueError, match="beta"):
            dot_amd.preference_loss(ratio.to(DEV), beta=beta)
    many = torch.zeros(1, device=DEV)
    with pytest.raises(ValueError, match="answers"):
        dot_amd.preference_loss(many.expand(2**23 + 2))
    with pytest.raises(ValueError, match="answers"):
        dot_amd.preference_loss(many.expand(2**22 + 2), plan=many.expand(1, 2**22 + 1))
