"""sequence_logp on the device against the float64 definition.

Tolerances.  A position's value is (x_a - m) k ln 2 - log s: the sum s of V
exponentials has a relative error below 2^-20 (each term: argument rounded
once, |d| 2^-24, hardware exponential 2^-23, partial sums of at most V / 256
terms; 1e-6), k = fl(log2 e / tau) is off by 2^-24 of |x_a - E_p[x]| / tau
(40 here at most: 2.4e-6).  So |error| <= 4e-6 per position, plus half a step
of fp32 of the result.  Gradients: c (delta - p), p to 4e-6 of itself, plus half
a step of the gradient's type; judged against the largest |c|.
"""

import numpy as np
import pytest
import torch

import dot_amd
from oracle import training as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
PER_POSITION = 4e-6
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def make(rng, B, S, V, dtype):
    x = torch.as_tensor((2 * rng.standard_normal((B, S, V))).astype(np.float32)).to(dtype)
    tokens = rng.integers(0, V, (B, S))
    for b in range(B):
        for s in range(S):
            x[b, s, tokens[b, s]] = float(np.log(V)) - 2 + 8 * rng.random()
    return x, tokens


def call(x, tokens, ref=None, mask=None, tau=1.0, reduction="sum", int_type=torch.int64):
    to = lambda a, t=None: None if a is None else torch.as_tensor(a, dtype=t).to(DEV)  # noqa: E731
    return dot_amd.sequence_logp(x, to(tokens, int_type), ref_logp=to(ref), mask=to(mask), tau=tau, reduction=reduction)


def check(logits, tokens, ref=None, mask=None, tau=1.0, reduction="sum", int_type=torch.int64, x=None, seed=0):
    dtype = logits.dtype
    x = logits.to(DEV) if x is None else x
    x = x.detach().requires_grad_()
    out = call(x, tokens, ref, mask, tau, reduction, int_type)
    o, p, weight = oracle.sequence_logp(logits.float().numpy(), tokens, ref, mask, tau, reduction)
    n = np.ones_like(o) if reduction == "none" else np.maximum((weight > 0).sum(1), 1)
    if reduction == "mean":
        n = np.ones_like(o)
    bound = PER_POSITION * n + 2.0**-24 * np.abs(o) + 2.0**-24 * PER_POSITION
    got = out.detach().cpu().double().numpy()
    assert out.dtype == torch.float32 and got.shape == o.shape
    assert (np.abs(got - o) <= bound).all(), np.abs(got - o).max()
    rng = np.random.default_rng(seed)
    up = rng.standard_normal(o.shape).astype(np.float32)
    (g,) = torch.autograd.grad([out], [x], [torch.as_tensor(up).to(DEV)])
    og = oracle.sequence_logp_grad(p, weight, tokens, up, tau)
    assert g.dtype == dtype and g.shape == x.shape
    half = 2.0**-24 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    tiny = 0 if dtype == torch.float32 else float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    c = np.abs((up if up.ndim == 2 else up[:, None]) * weight / tau)[:, :, None]
    err = np.abs(g.detach().cpu().double().numpy() - og)
    # at the taken token c and c p cancel: the error stays one of c
    assert (err <= (half + 8e-6) * np.abs(og) + 2e-6 * c + tiny).all(), (err - (half + 8e-6) * np.abs(og)).max()
    assert (g[torch.as_tensor(weight == 0).to(DEV)] == 0).all()
    return out.detach(), g


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 64, 255, 1000, 2048, 4099, 32768])
def test_vocabularies(dtype, V):
    print(f"[logp] {dtype} V={V}", flush=True)
    rng = np.random.default_rng(V)
    logits, tokens = make(rng, 2, 5, V, DTYPES[dtype])
    check(logits, tokens)
    check(logits, tokens, tau=0.6, reduction="none")


@pytest.mark.parametrize("B,S,V", [(1, 1, 100003), (1, 1, 131072), (3, 17, 50021), (1, 300, 4000), (40, 70, 64)])
@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
def test_lengths(B, S, V, reduction):
    print(f"[logp] B={B} S={S} V={V} {reduction}", flush=True)
    rng = np.random.default_rng(S)
    logits, tokens = make(rng, B, S, V, torch.bfloat16)
    ref = (-3 * rng.random((B, S))).astype(np.float32)
    mask = rng.random((B, S)) < 0.7
    mask[0, 0] = True
    if B > 1:
        mask[1] = False  # a sequence without positions
    check(logits, tokens, ref=ref, mask=mask, tau=1.3, reduction=reduction)


@pytest.mark.parametrize("ref_type", [np.float32, np.float64])
@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("int_type", [torch.int32, torch.int64])
def test_references(ref_type, per_token, int_type):
    rng = np.random.default_rng(1)
    logits, tokens = make(rng, 3, 20, 500, torch.float32)
    o, _, _ = oracle.sequence_logp(logits.numpy(), tokens, reduction="none" if per_token else "sum")
    ref = (o + 0.1 * rng.standard_normal(o.shape)).astype(ref_type)
    check(logits, tokens, ref=ref, int_type=int_type)
    check(logits, tokens, ref=ref, reduction="mean", int_type=int_type)


@pytest.mark.parametrize("tau", [1.0, 1.3, 0.7])
def test_long_sum_keeps_its_digits(tau):
    """The log ratio of a long answer to a reference given per position: a few units out of thousands."""
    rng = np.random.default_rng(2)
    logits, tokens = make(rng, 2, 4096, 300, torch.float32)
    per, _, _ = oracle.sequence_logp(logits.numpy(), tokens, tau=tau, reduction="none")
    ref = per + 1e-3 * rng.standard_normal(per.shape)
    want, _, _ = oracle.sequence_logp(logits.numpy(), tokens, ref=ref, tau=tau)
    got = call(logits.to(DEV), tokens, ref=ref, tau=tau).cpu().double().numpy()
    assert (np.abs(got - want) <= 4096 * PER_POSITION).all()
    # Errors of single positions have both signs: 1e-7 sqrt(4096) is 6e-6, and 5e-8 of bias 2e-4.  A temperature
    # rounded to fp32 would give 4e-8 of x - E[x], 6e-4 here; sums in fp32 are off by 4e-3.
    assert np.abs(got - want).max() < 3e-4


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_likely_tokens_keep_their_digits(dtype):
    """The value of a token that is nearly certain is small: its error is relative to it (and half a step of fp32).

    sum of the others / own: each term to 2^-22, their sum to 2^-21 of itself, so 1e-6 of log(1 + that)."""
    rng = np.random.default_rng(9)
    for V in (8, 100, 4099, 40000):
        x = torch.as_tensor(rng.standard_normal((2, 9, V)).astype(np.float32))
        tokens = rng.integers(0, V, (2, 9))
        for s in range(9):
            x[:, s].scatter_(1, torch.as_tensor(tokens[:, s])[:, None], 12.0 + 2 * s)
        x = x.to(DTYPES[dtype])
        got = call(x.to(DEV), tokens, reduction="none").cpu().double().numpy()
        want = torch.log_softmax(x.double(), -1).numpy()[np.arange(2)[:, None], np.arange(9)[None], tokens]
        # log_softmax in 64 bits is itself off by 1e-15 of the largest logit
        assert (np.abs(got - want) <= 2e-6 * np.abs(want) + 1e-14).all()


def test_tokens_outside_are_left_out():
    rng = np.random.default_rng(3)
    logits, tokens = make(rng, 2, 12, 77, torch.bfloat16)
    tokens[0, 3], tokens[0, 4], tokens[1, 0], tokens[1, 1] = -100, 77, 2**32, -1
    for reduction in ("sum", "mean", "none"):
        check(logits, tokens, reduction=reduction)


def test_left_out_positions_are_not_read():
    rng = np.random.default_rng(4)
    for V in (64, 301, 5000):
        logits, tokens = make(rng, 2, 16, V, torch.float32)
        mask = rng.random((2, 16)) < 0.5
        dirty = logits.clone()
        dirty[~torch.as_tensor(mask)] = float("nan")
        a = check(logits, tokens, mask=mask)
        x = dirty.to(DEV).requires_grad_()
        out = call(x, tokens, mask=mask)
        (g,) = torch.autograd.grad(out.sum(), x)
        assert torch.equal(out, a[0]) and torch.isfinite(g).all()


def test_masked_vocabulary():
    """Logits of -inf and of the type's lowest value, a row of nothing else, a certain token."""
    rng = np.random.default_rng(5)
    for dtype in DTYPES.values():
        logits, tokens = make(rng, 1, 6, 90, dtype)
        keep = {int(t) for t in tokens[0]}
        others = [v for v in range(90) if v not in keep]
        logits[0, 0, others] = -float("inf")
        logits[0, 1, others] = torch.finfo(dtype).min
        logits[0, 2] = torch.finfo(dtype).min  # log of 1 / 90
        logits[0, 3] = -float("inf")
        logits[0, 3, tokens[0, 3]] = 1.0       # certain: 0
        logits[0, 4] = torch.finfo(dtype).min
        logits[0, 4, tokens[0, 4]] = 100.0
        out, g = check(logits, tokens, reduction="none")
        assert out[0, 3] == 0 and (g[0, 3] == 0).all() and abs(float(out[0, 2]) + np.log(90)) < 1e-5
    # a token that cannot be: -inf, as log_softmax gives
    logits[0, 5, tokens[0, 5]] = -float("inf")
    out = call(logits.to(DEV), tokens, reduction="none")
    assert out[0, 5] == -float("inf")
    # NaN and +inf show at their position alone
    logits[0, 1, 5] = float("nan")
    logits[0, 2, 5] = float("inf")
    out = call(logits.to(DEV), tokens, reduction="none")
    assert torch.isnan(out[0]).tolist() == [False, True, True, False, False, False]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype):
    """Shifted views, odd offsets and strides of the logits; other layouts of tokens and masks; no batch dimension."""
    rng = np.random.default_rng(6)
    logits, tokens = make(rng, 4, 11, 520, DTYPES[dtype])
    views = {
        "shifted": (lambda t: t[:, :-1], slice(None), slice(0, 10)),
        "offset": (lambda t: t[:, :, 3:503], slice(None), slice(None)),
        "odd rows": (lambda t: t[::2, 1::2, 1:], slice(0, 4, 2), slice(1, 11, 2)),
        "broadcast": (lambda t: t[:1].expand(4, 11, 520), slice(None), slice(None)),
        "columns": (lambda t: t[:, :, ::3], slice(None), slice(None)),
    }
    for name, (view, bs, ss) in views.items():
        print(f"[logp] {dtype} {name}", flush=True)
        v = view(logits)
        tk = tokens[bs, ss] % v.shape[2]
        x = view(logits.to(DEV))
        assert not x.is_contiguous()
        check(v.contiguous(), tk, x=x)
    strided = torch.as_tensor(np.repeat(tokens, 2, 1)).to(DEV)[:, ::2]
    mask = torch.ones(11, 4, dtype=torch.bool, device=DEV).t()
    a = dot_amd.sequence_logp(logits.to(DEV), strided, mask=mask)
    b = call(logits.to(DEV), tokens)
    assert torch.equal(a, b)
    one = dot_amd.sequence_logp(logits[2].to(DEV), torch.as_tensor(tokens[2]).to(DEV), ref_logp=torch.tensor(1.0, device=DEV))
    assert one.shape == () and abs(float(one) - (float(b[2]) - 1.0)) <= 2.0**-22 * abs(float(b[2]))
    per = dot_amd.sequence_logp(logits[2].to(DEV), torch.as_tensor(tokens[2]).to(DEV), reduction="none")
    assert per.shape == (11,)


def test_expanded_gradient():
    """The gradient of a sum is an expanded scalar; it equals the written-out one."""
    rng = np.random.default_rng(7)
    logits, tokens = make(rng, 3, 9, 333, torch.bfloat16)
    for reduction in ("sum", "none"):
        x = logits.to(DEV).requires_grad_()
        out = call(x, tokens, reduction=reduction)
        (a,) = torch.autograd.grad(out.sum(), x, retain_graph=True)
        (b,) = torch.autograd.grad([out], [x], [torch.ones_like(out)])
        assert torch.equal(a, b)


def test_empty():
    for B, S in ((0, 4), (3, 0), (0, 0)):
        x = torch.zeros(B, S, 10, device=DEV, requires_grad=True)
        tokens = torch.zeros(B, S, dtype=torch.int64, device=DEV)
        out = dot_amd.sequence_logp(x, tokens, ref_logp=torch.ones(B, device=DEV))
        assert out.shape == (B,) and (out == -1).all()
        assert dot_amd.sequence_logp(x, tokens, reduction="none").shape == (B, S)
        (g,) = torch.autograd.grad(out.sum(), x)
        assert g.shape == x.shape


def test_large_offsets():
    """Rows beyond 2^31 elements: the last rows of a large tensor, and the same bits twice."""
    B, S, V = 5, 1024, 500000
    x = torch.empty(B, S, V, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(0))
    tokens = torch.randint(0, V, (B, S), device=DEV)
    mask = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    mask[0, 0] = mask[2, 700] = mask[4, 1022:] = True
    x.requires_grad_()
    out = dot_amd.sequence_logp(x, tokens, mask=mask, reduction="none")
    (g,) = torch.autograd.grad(out.sum(), x)
    (g2,) = torch.autograd.grad(dot_amd.sequence_logp(x, tokens, mask=mask, reduction="none").sum(), x)
    out = out.detach()
    for b, s in ((0, 0), (2, 700), (4, 1022), (4, 1023)):
        row = x[b, s].detach().double()
        want = torch.log_softmax(row, 0)
        t = int(tokens[b, s])
        assert abs(float(out[b, s]) - float(want[t])) <= PER_POSITION + 2.0**-23 * abs(float(want[t]))
        og = -torch.exp(want)
        og[t] += 1
        assert (g[b, s].double() - og).abs().max() <= 2.0**-8 + 1e-5
        assert torch.equal(g[b, s], g2[b, s])
    assert int((g[1] != 0).sum()) == 0 and int((g[4, :1022] != 0).sum()) == 0


def test_other_stream_and_graph():
    rng = np.random.default_rng(8)
    data = [make(rng, 2, 33, 3000, torch.bfloat16) for _ in range(3)]
    data = [(x.to(DEV), torch.as_tensor(t).to(DEV)) for x, t in data]

    def step(logits, tokens):
        x = logits.detach().requires_grad_()
        out = dot_amd.sequence_logp(x, tokens)
        (g,) = torch.autograd.grad(out.sum(), x)
        return out.detach(), g

    eager = [step(*d) for d in data]
    hx, ht = data[0][0].clone(), data[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(hx, ht)
        step(hx, ht)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, eager[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(hx, ht)
    for i in (1, 2, 0, 2):
        hx.copy_(data[i][0])
        ht.copy_(data[i][1])
        graph.replay()
        torch.cuda.synchronize()
        between = step(*data[(i + 1) % 3])
        assert all(torch.equal(a, b) for a, b in zip(outs, eager[i]))
        assert all(torch.equal(a, b) for a, b in zip(between, eager[(i + 1) % 3]))
