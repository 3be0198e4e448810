"""distill_loss on the device against the float64 definition; tolerances in generation_cases.py."""

import numpy as np
import pytest
import torch

import dot_amd
from generation_cases import DTYPES, SUM, array, check_distill, logits_of, teacher_of
from oracle import generation as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FORMS = [("forward", "bucket"), ("forward", "none"), ("reverse", "bucket")]


def check(logits, logp, tokens, int_type=torch.int32, x=None, **kw):
    lp, tk = torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens, dtype=int_type).to(DEV)

    def call(x, mask, **kw):
        mask = None if mask is None else torch.as_tensor(mask).to(DEV)
        return dot_amd.distill_loss(x, lp, tk, mask=mask, **kw)

    return check_distill(call, logits, logp, tokens, x=logits.to(DEV) if x is None else x, **kw)


@pytest.mark.parametrize("direction,rest", FORMS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [2, 7, 8, 9, 63, 64, 255, 1000, 2048, 4099, 32768])
def test_vocabularies(dtype, V, direction, rest):
    print(f"[distill] {dtype} V={V} {direction} {rest}", flush=True)
    rng = np.random.default_rng(V)
    logits = logits_of(rng, (2, 3, V), DTYPES[dtype])
    for k in sorted({1, min(V - 1, 5), min(V - 1, 64)}):
        logp, tokens = teacher_of(rng, logits, k)
        check(logits, logp, tokens, direction=direction, rest=rest)
    logp, tokens = teacher_of(rng, logits, min(V - 1, 100), tau=0.7)
    check(logits, logp, tokens, tau=0.7, reduction="none", direction=direction, rest=rest)


@pytest.mark.parametrize("direction,rest", FORMS)
@pytest.mark.parametrize("B,S,V,k", [(1, 1, 100003, 200), (1, 1, 131072, 64), (3, 17, 50021, 33), (1, 300, 4000, 20),
                                     (40, 70, 64, 8), (1, 2, 600000, 256)])
@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
def test_lengths(B, S, V, k, reduction, direction, rest):
    print(f"[distill] B={B} S={S} V={V} k={k} {reduction} {direction} {rest}", flush=True)
    rng = np.random.default_rng(S)
    logits = logits_of(rng, (B, S, V), torch.bfloat16)
    logp, tokens = teacher_of(rng, logits, k, tau=1.3)
    mask = rng.random((B, S)) < 0.7
    mask[0, 0] = True
    if B > 1:
        mask[1] = False  # a sequence without positions
    check(logits, logp, tokens, mask=mask, tau=1.3, reduction=reduction, direction=direction, rest=rest,
          int_type=torch.int64 if S % 2 else torch.int32)


@pytest.mark.parametrize("direction,rest", FORMS)
@pytest.mark.parametrize("V", [50, 3000, 300000])
def test_entries_that_name_no_token(V, direction, rest):
    """Tokens outside, named twice (the first counts) or with a log-probability of -inf; positions without any."""
    rng = np.random.default_rng(V)
    logits = logits_of(rng, (2, 5, V), torch.float32)
    logp, tokens = teacher_of(rng, logits, 12)
    tokens[0, 0, 3], tokens[0, 0, 4], tokens[0, 1, 0], tokens[1, 0, 11] = -100, V, 2**32 + 1, -1
    tokens[0, 2, 5:8] = tokens[0, 2, 2]
    tokens[0, 3, 0] = tokens[0, 3, 11]
    logp[0, 4, 6:] = -np.inf
    logp[1, 1, 0] = -np.inf
    tokens[1, 1, 5] = tokens[1, 1, 0]   # named by a later entry after all
    tokens[1, 2] = -1
    logp[1, 3] = -np.inf
    tokens[1, 4] = tokens[1, 4, :1]     # one token
    for reduction in ("sum", "mean", "none"):
        check(logits, logp, tokens, reduction=reduction, int_type=torch.int64, direction=direction, rest=rest)


@pytest.mark.parametrize("direction,rest", FORMS)
def test_left_out_positions_are_not_read(direction, rest):
    rng = np.random.default_rng(4)
    for V in (64, 301, 5000, 70000):
        logits = logits_of(rng, (2, 6, V), torch.float32)
        logp, tokens = teacher_of(rng, logits, 8)
        mask = rng.random((2, 6)) < 0.5
        tokens[0, 0] = -1
        mask[0, 0] = True
        gone = ~torch.as_tensor(mask)
        gone[0, 0] = True
        dirty = logits.clone()
        dirty[gone] = float("nan")
        kw = dict(direction=direction, rest=rest)
        a = check(logits, logp, tokens, mask=mask, **kw)
        x = dirty.to(DEV).requires_grad_()
        out = dot_amd.distill_loss(x, torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens).to(DEV),
                                   mask=torch.as_tensor(mask).to(DEV), **kw)
        (g,) = torch.autograd.grad(out.sum(), x)
        assert torch.equal(out, a[0]) and torch.isfinite(g).all() and (g[gone.to(DEV)] == 0).all()


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_vocabulary(dtype):
    """Logits of -inf and of the type's lowest value among the teacher's tokens and the others."""
    rng = np.random.default_rng(5)
    low = torch.finfo(DTYPES[dtype]).min
    for V in (90, 3000):
        logits = logits_of(rng, (1, 7, V), DTYPES[dtype])
        logp, tokens = teacher_of(rng, logits, 6)
        named = torch.zeros(7, V, dtype=torch.bool)
        named.scatter_(1, torch.as_tensor(tokens[0]), True)
        logits[0, 0][~named[0]] = -float("inf")   # no other token: the teacher's rest has no place
        logits[0, 1][~named[1]] = low
        logits[0, 2, tokens[0, 2, 1]] = -float("inf")
        logits[0, 3] = low
        logits[0, 4][named[4]] = low              # the teacher's tokens are out of reach
        logits[0, 5] = -float("inf")
        logits[0, 5, tokens[0, 5, 0]] = 1.0       # certain
        for direction, rest in FORMS:
            keep = [0, 1, 2, 3, 4, 5, 6]
            out, g = check(logits[:, keep], logp[:, keep], tokens[:, keep], reduction="none", direction=direction, rest=rest)
            assert torch.isfinite(g).all()
            assert (out[0, 0] == float("inf")) == ((direction, rest) == ("forward", "bucket"))
            assert out[0, 2] == float("inf") or direction == "reverse"
    # the teacher's rest is rounding alone: not held against a student that allows no other token
    logp = np.log(np.array([[[0.75, 0.25]]])).astype(np.float32)
    logits = torch.full((1, 1, 5), -float("inf"))
    logits[0, 0, 1], logits[0, 0, 3] = 2.0, 1.0
    out, _ = check(logits.to(DTYPES[dtype]), logp, np.array([[[1, 3]]]))
    assert torch.isfinite(out).all()


def test_nan_shows_at_its_position_alone():
    rng = np.random.default_rng(6)
    logits = logits_of(rng, (1, 6, 200), torch.float32)
    logp, tokens = teacher_of(rng, logits, 5)
    other = [v for v in range(200) if v not in set(tokens[0].ravel().tolist())][0]
    logits[0, 1, other] = float("nan")
    logits[0, 2, tokens[0, 2, 0]] = float("inf")
    logits[0, 3, tokens[0, 3, 1]] = float("nan")
    logp[0, 4, 2] = np.nan
    for direction, rest in FORMS:
        x = logits.to(DEV).requires_grad_()
        out = dot_amd.distill_loss(x, torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens).to(DEV), reduction="none",
                                   direction=direction, rest=rest)
        (g,) = torch.autograd.grad(out.sum(), x)
        assert torch.isnan(out[0]).tolist() == [False, True, True, True, True, False]
        assert torch.isnan(g[0]).any(-1).tolist() == [False, True, True, True, True, False]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype):
    rng = np.random.default_rng(7)
    logits = logits_of(rng, (4, 11, 520), DTYPES[dtype])
    views = {
        "shifted": lambda t: t[:, :-1],
        "offset": lambda t: t[:, :, 3:503],
        "odd rows": lambda t: t[::2, 1::2, 1:],
        "broadcast": lambda t: t[:1].expand(4, 11, 520),
        "columns": lambda t: t[:, :, ::3],
    }
    for name, view in views.items():
        print(f"[distill] {dtype} {name}", flush=True)
        v = view(logits).contiguous()
        logp, tokens = teacher_of(rng, v, 9)
        check(v, logp, tokens, x=view(logits.to(DEV)))
    # other layouts and types of the teacher's part and the mask; no batch dimension
    logp, tokens = teacher_of(rng, logits, 9)
    a, _ = check(logits, logp, tokens)
    lp, tk = torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens).to(DEV)
    mask = torch.ones(11, 4, dtype=torch.bool, device=DEV).t()
    b = dot_amd.distill_loss(logits.to(DEV), lp.double().transpose(0, 2).contiguous().transpose(0, 2),
                             tk.repeat_interleave(2, -1)[..., ::2], mask=mask)
    assert torch.equal(a, b)
    one = dot_amd.distill_loss(logits[2].to(DEV), lp[2], tk[2])
    assert one.shape == () and torch.equal(one, a[2])
    assert dot_amd.distill_loss(logits[2].to(DEV), lp[2], tk[2], reduction="none").shape == (11,)


def test_small_divergences_keep_their_digits():
    """A student next to its teacher: the loss is a small difference of log-probabilities.

    Forwards its slope by the others' sum is Q_r - P_r, which is as small: what is left is the teacher's fp32."""
    rng = np.random.default_rng(8)
    logits = logits_of(rng, (2, 9, 5000), torch.float32)
    logp, tokens = teacher_of(rng, logits, 32, noise=1e-3)
    lp, tk = torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens).to(DEV)
    got = array(dot_amd.distill_loss(logits.to(DEV), lp, tk, reduction="none"))
    want, parts = oracle.distill(array(logits), logp, tokens, reduction="none")
    slope = np.array([[abs(parts[b, s]["other"]) for s in range(9)] for b in range(2)])
    assert np.abs(want).max() < 1e-4
    assert (np.abs(got - want) <= SUM * slope + 2.0**-24 * np.abs(want) + 1e-12).all()


def test_likely_tokens_keep_their_digits():
    """Gradients where teacher and student agree on a nearly certain token: differences of numbers next to 1."""
    rng = np.random.default_rng(9)
    x = torch.as_tensor(rng.standard_normal((1, 8, 4099)).astype(np.float32))
    x[..., 17] = 22.0
    logp, tokens = teacher_of(rng, x, 4, noise=0.3)
    _, parts = oracle.distill(array(x), logp, tokens, reduction="none")
    leaf = x.to(DEV).requires_grad_()
    out = dot_amd.distill_loss(leaf, torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens).to(DEV), reduction="none")
    (g,) = torch.autograd.grad(out.sum(), leaf)
    for s in range(8):
        p = parts[0, s]
        # Q (1 - Q) SUM of the token itself, and half a step
        bound = SUM * p["Q"][17] * (1 - p["Q"][17]) + 2.0**-23 * abs(p["pull"][17]) + 1e-15
        assert abs(float(g[0, s, 17]) - p["pull"][17]) <= bound


def test_far_likelier_named_tokens():
    """The others' exponentials relative to the named token's are below the smallest float: their shares are not."""
    rng = np.random.default_rng(10)
    x = torch.as_tensor(rng.standard_normal((1, 4, 600)).astype(np.float32))
    x[..., 3] = 200.0
    logp = np.log(np.full((1, 4, 1), 0.5)).astype(np.float32)
    tokens = np.full((1, 4, 1), 3)
    for direction, rest in FORMS:
        out, g = check(x, logp, tokens, direction=direction, rest=rest, reduction="none")
        assert torch.isfinite(out).all() and torch.isfinite(g).all()
        if (direction, rest) == ("forward", "bucket"):
            assert abs(float(g[0, 0].sum())) < 1e-5 and float(g[0, 0, 3]) > 0.49


def test_expanded_gradient():
    rng = np.random.default_rng(11)
    logits = logits_of(rng, (3, 9, 333), torch.bfloat16)
    logp, tokens = teacher_of(rng, logits, 7)
    lp, tk = torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens).to(DEV)
    for reduction in ("sum", "mean", "none"):
        x = logits.to(DEV).requires_grad_()
        out = dot_amd.distill_loss(x, lp, tk, reduction=reduction)
        (a,) = torch.autograd.grad(out.sum(), x, retain_graph=True)
        (b,) = torch.autograd.grad([out], [x], [torch.ones_like(out)])
        assert torch.equal(a, b)
        assert torch.equal(dot_amd.distill_loss(x.detach(), lp, tk, reduction=reduction), out)


def test_empty():
    for B, S in ((0, 4), (3, 0), (0, 0)):
        x = torch.zeros(B, S, 10, device=DEV, requires_grad=True)
        lp, tk = torch.zeros(B, S, 2, device=DEV), torch.zeros(B, S, 2, dtype=torch.int64, device=DEV)
        out = dot_amd.distill_loss(x, lp, tk)
        assert out.shape == (B,) and (out == 0).all()
        assert dot_amd.distill_loss(x, lp, tk, reduction="none").shape == (B, S)
        (g,) = torch.autograd.grad(out.sum(), x)
        assert g.shape == x.shape


def test_large_offsets():
    """Rows beyond 2^31 elements, and the same bits twice."""
    B, S, V, K = 5, 1024, 500000, 40
    x = torch.empty(B, S, V, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(0))
    mask = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    at = ((0, 0), (2, 700), (4, 1022), (4, 1023))
    for b, s in at:
        mask[b, s] = True
    rng = np.random.default_rng(0)
    rows = torch.stack([x[b, s] for b, s in at]).cpu()[None]
    logp, tokens = teacher_of(rng, rows, K)
    lp, tk = torch.zeros(B, S, K, device=DEV), torch.zeros(B, S, K, dtype=torch.int32, device=DEV)
    for i, (b, s) in enumerate(at):
        lp[b, s], tk[b, s] = torch.as_tensor(logp[0, i]).to(DEV), torch.as_tensor(tokens[0, i]).to(DEV)
    x.requires_grad_()
    out = dot_amd.distill_loss(x, lp, tk, mask=mask, reduction="none")
    (g,) = torch.autograd.grad(out.sum(), x)
    (g2,) = torch.autograd.grad(dot_amd.distill_loss(x, lp, tk, mask=mask, reduction="none").sum(), x)
    want, parts = oracle.distill(array(rows), logp, tokens, reduction="none")
    for i, (b, s) in enumerate(at):
        assert abs(float(out[b, s]) - want[0, i]) <= SUM + 2.0**-23 * abs(want[0, i])
        pull = parts[0, i]["pull"]
        assert (np.abs(array(g[b, s]) - pull) <= (2.0**-8 + 1e-5) * np.abs(pull) + 3 * SUM * parts[0, i]["Q"] + 1e-37).all()
        assert torch.equal(g[b, s], g2[b, s])
    assert int((g[1] != 0).sum()) == 0 and int((g[4, :1022] != 0).sum()) == 0


def test_other_stream_and_graph():
    rng = np.random.default_rng(12)
    data = []
    for _ in range(3):
        x = logits_of(rng, (2, 33, 3000), torch.bfloat16)
        logp, tokens = teacher_of(rng, x, 30)
        data.append((x.to(DEV), torch.as_tensor(logp).to(DEV), torch.as_tensor(tokens).to(DEV)))

    def step(logits, logp, tokens):
        x = logits.detach().requires_grad_()
        out = dot_amd.distill_loss(x, logp, tokens)
        (g,) = torch.autograd.grad(out.sum(), x)
        return out.detach(), g

    eager = [step(*d) for d in data]
    held = [t.clone() for t in data[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*held)
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, eager[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*held)
    for i in (1, 2, 0, 2):
        for h, d in zip(held, data[i]):
            h.copy_(d)
        graph.replay()
        torch.cuda.synchronize()
        between = step(*data[(i + 1) % 3])
        assert all(torch.equal(a, b) for a, b in zip(outs, eager[i]))
        assert all(torch.equal(a, b) for a, b in zip(between, eager[(i + 1) % 3]))
