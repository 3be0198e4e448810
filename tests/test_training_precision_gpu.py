"""Digits of the routing, sequence log-probability and preference operators on the
device, element by element against the float64 definition."""

import pytest
import torch

import dot_amd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def half_step(dtype):
    """Relative, and absolute for results that are subnormal."""
    info = torch.finfo(dtype)
    return info.eps / 2, float(info.smallest_normal) * info.eps / 2


def test_gradient_of_large_logits():
    """Rows beyond 2^31 elements, before and behind where the caches end, every entry to half a step: p is good to 5e-6
    of itself (see above; logits up to 19 below the largest)."""
    B, S, V = 5, 1024, 500000
    x = torch.empty(B, S, V, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(0))
    tokens = torch.randint(0, V, (B, S), device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    # the last 224 MB, 234 rows of 10^6 bytes, are read through the caches: rows from 4886 on
    rows = [(0, 0), (2, 700), (4, 789), (4, 790), (4, 1022), (4, 1023)]
    mask = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    large = [0, 1, 7, 8, V // 3, V // 2 - 1, V // 2, V - 9, V - 8, V - 1]
    for i, (b, s) in enumerate(rows):
        mask[b, s] = True
        x[b, s, large] = 10.0 + torch.arange(len(large), device=DEV).roll(i).bfloat16() / 4
        tokens[b, s] = (large + [int(tokens[b, s])])[2 * i]
    x.requires_grad_()
    out = dot_amd.sequence_logp(x, tokens, mask=mask, reduction="none")
    (g,) = torch.autograd.grad(out.sum(), x)
    half, tiny = half_step(torch.bfloat16)
    for b, s in rows:
        want = -torch.softmax(x[b, s].detach().double(), 0)
        t = int(tokens[b, s])
        want[t] += 1
        assert want[large].abs().min() > 1e-3
        assert ((g[b, s].double() - want).abs() <= (half + 5e-6) * want.abs() + tiny).all(), (b, s)
    g[mask] = 0
    assert not g.any()
