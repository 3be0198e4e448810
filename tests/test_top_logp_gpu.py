"""top_logp on the device against the float64 definition; tolerances in generation_cases.py."""

import numpy as np
import pytest
import torch

import dot_amd
from generation_cases import DTYPES, check_top, logits_of

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def check(logits, k, tau=1.0, mask=None, x=None):
    x = logits.to(DEV) if x is None else x
    r = dot_amd.top_logp(x, k, tau=tau, mask=None if mask is None else torch.as_tensor(mask).to(DEV))
    check_top(r, logits, k, tau, mask)
    return r


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 64, 255, 1000, 2048, 2049, 4099, 32768])
def test_vocabularies(dtype, V):
    print(f"[top] {dtype} V={V}", flush=True)
    rng = np.random.default_rng(V)
    logits = logits_of(rng, (2, 3, V), DTYPES[dtype])
    for k in sorted({1, min(V, 5), min(V, 64), min(V, 65), min(V, 256)}):
        check(logits, k, tau=0.7 if k % 2 else 1.0)


@pytest.mark.parametrize("B,S,V,k", [(1, 1, 100003, 200), (1, 1, 131072, 64), (3, 17, 50021, 33), (600, 1, 4000, 20),
                                     (2, 3, 160001, 256), (40, 30, 20000, 128), (1, 2, 400000, 100)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_lengths(B, S, V, k, dtype):
    print(f"[top] {dtype} B={B} S={S} V={V} k={k}", flush=True)
    rng = np.random.default_rng(S)
    logits = logits_of(rng, (B, S, V), DTYPES[dtype])
    mask = rng.random((B, S)) < 0.8
    mask[0, 0] = True
    check(logits, k, tau=2.0, mask=mask)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [300, 5000, 40000])
@pytest.mark.parametrize("kind", ["equal", "two", "coarse", "ascending", "descending", "one thread", "zeros"])
def test_orders(dtype, V, kind):
    """Rows of equal logits and orders in which the largest ones lie together, or all 2048 or 1024 apart."""
    print(f"[top] {dtype} V={V} {kind}", flush=True)
    rng = np.random.default_rng(V)
    at = np.arange(V)
    row = {
        "equal": np.full(V, 1.5),
        "two": np.where(rng.random(V) < 0.5, -1.0, 2.0),
        "coarse": np.round(2 * rng.standard_normal(V)),
        "ascending": at / V * 20 - 10,
        "descending": 10 - at / V * 20,
        "one thread": np.where(at % 2048 == 8, 5.0, 0.0) + np.where(at % 1024 == 4, 2.0, 0.0) + 0.01 * rng.random(V),
        "zeros": np.where(rng.random(V) < 0.5, -0.0, 0.0),
    }[kind]
    logits = torch.as_tensor(np.stack([row, row[::-1].copy()]).astype(np.float32))[None].to(DTYPES[dtype])
    for k in (1, 20, 64, 100, 256):
        check(logits, min(k, V))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_masked_vocabulary(dtype):
    """Logits of -inf and of the type's lowest value, rows with fewer than k others, NaN and +inf."""
    rng = np.random.default_rng(1)
    for V in (40, 3000, 70000):
        logits = logits_of(rng, (1, 8, V), DTYPES[dtype])
        low = torch.finfo(DTYPES[dtype]).min
        some = rng.choice(V, 30, replace=False)
        keep = torch.zeros(V, dtype=torch.bool)
        keep[torch.as_tensor(some)] = True
        logits[0, 0, ~keep] = -float("inf")
        logits[0, 1, ~keep] = low
        logits[0, 2] = -float("inf")
        logits[0, 3] = low
        logits[0, 4, ~keep] = low
        logits[0, 4, keep] = -float("inf")
        logits[0, 5, int(some[0])] = float("nan")
        logits[0, 6, int(some[1])] = float("inf")
        logits[0, 7] = float("nan")
        for k in (5, 31, min(V, 200)):
            r = check(logits, k)
            assert (r.tokens[0, 2] == -1).all() and (r.tokens[0, 7] == -1).all()
            assert torch.isnan(r.logp[0, 5, :5]).all() and r.tokens[0, 6, 0] == int(some[1])


def test_left_out_positions_are_not_read():
    rng = np.random.default_rng(2)
    for V, k in ((64, 8), (5000, 40), (70000, 100)):
        logits = logits_of(rng, (2, 6, V), torch.float32)
        mask = rng.random((2, 6)) < 0.5
        dirty = logits.clone()
        dirty[~torch.as_tensor(mask)] = float("nan")
        a = check(logits, k, mask=mask)
        b = dot_amd.top_logp(dirty.to(DEV), k, mask=torch.as_tensor(mask).to(DEV))
        assert torch.equal(a.logp, b.logp) and torch.equal(a.tokens, b.tokens)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype):
    rng = np.random.default_rng(3)
    logits = logits_of(rng, (4, 11, 520), DTYPES[dtype])
    views = {
        "shifted": lambda t: t[:, :-1],
        "offset": lambda t: t[:, :, 3:503],
        "odd rows": lambda t: t[::2, 1::2, 1:],
        "broadcast": lambda t: t[:1].expand(4, 11, 520),
        "columns": lambda t: t[:, :, ::3],
        "transposed": lambda t: t.transpose(0, 1),
    }
    for name, view in views.items():
        print(f"[top] {dtype} {name}", flush=True)
        check(view(logits).contiguous(), 17, x=view(logits.to(DEV)))
    one = dot_amd.top_logp(logits[2].to(DEV), 9, mask=torch.ones(11, dtype=torch.bool, device=DEV))
    all_ = dot_amd.top_logp(logits.to(DEV), 9)
    assert torch.equal(one.logp, all_.logp[2]) and torch.equal(one.tokens, all_.tokens[2])


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_equal_rows_have_equal_bits_wherever_they_lie(dtype):
    rng = np.random.default_rng(4)
    for V in (1001, 33333):
        row = logits_of(rng, (1, V), DTYPES[dtype])[0].to(DEV)
        flat = torch.zeros(12 * (V + 3), dtype=row.dtype, device=DEV)
        x = flat[1 : 1 + 10 * (V + 3)].view(10, V + 3)[:, :V]
        x[:] = row
        r = dot_amd.top_logp(x, 50)
        assert (r.logp == r.logp[:1]).all() and (r.tokens == r.tokens[:1]).all()


@pytest.mark.parametrize("V", [2, 40000])
@pytest.mark.parametrize("tau", [0.7, 1.0, 1.3])
def test_logits_are_scaled_in_fp32(tau, V):
    """Each scaled logit and the difference from the largest one take a rounding of fp32, as in a program that scales
    its logits so: beams are compared by what these differences are.  Next to a logit of 100 the others' terms are
    below 2^-53 of its own, so that log-probabilities are the differences themselves."""
    rng = np.random.default_rng(6)
    x = np.full((300, V), -np.inf, np.float32)
    x[:, 0] = 100.0
    x[:, V - 1] = 40 + 5 * rng.random(300)
    inv = np.float32(1) / np.float32(tau)
    want = x[:, V - 1] * inv - x[:, 0] * inv
    assert want.dtype == np.float32
    r = dot_amd.top_logp(torch.as_tensor(x).to(DEV), 2, tau=tau)
    assert (r.tokens[:, 1] == V - 1).all() and np.array_equal(r.logp[:, 1].cpu().numpy(), want)


def test_empty():
    for B, S in ((0, 4), (3, 0), (0, 0)):
        r = dot_amd.top_logp(torch.zeros(B, S, 10, device=DEV), 3)
        assert r.logp.shape == (B, S, 3) and r.tokens.shape == (B, S, 3)


def test_large_offsets():
    """Rows beyond 2^31 elements, and the same bits twice."""
    B, S, V = 5, 1024, 500000
    x = torch.empty(B, S, V, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(0))
    mask = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    mask[0, 0] = mask[2, 700] = mask[4, 1022:] = True
    r, again = dot_amd.top_logp(x, 100, mask=mask), dot_amd.top_logp(x, 100, mask=mask)
    assert torch.equal(r.logp, again.logp) and torch.equal(r.tokens, again.tokens)
    at = ((0, 0), (2, 700), (4, 1022), (4, 1023))
    rows = torch.stack([x[b, s] for b, s in at]).cpu()[None]
    got = dot_amd.distillation.TopLogpResult(torch.stack([r.logp[i] for i in at])[None],
                                             torch.stack([r.tokens[i] for i in at])[None])
    check_top(got, rows, 100)
    assert int((r.tokens >= 0).sum()) == 4 * 100


def test_other_stream_and_graph():
    rng = np.random.default_rng(5)
    data = [logits_of(rng, (2, 33, 40000), torch.bfloat16).to(DEV) for _ in range(3)]
    step = lambda x: dot_amd.top_logp(x, 70, tau=1.5)  # noqa: E731
    same = lambda a, b: torch.equal(a.logp, b.logp) and torch.equal(a.tokens, b.tokens)  # noqa: E731
    eager = [step(x) for x in data]
    held = data[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(held)
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    assert same(other, eager[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for i in (1, 2, 0, 2):
        held.copy_(data[i])
        graph.replay()
        torch.cuda.synchronize()
        between = step(data[(i + 1) % 3])
        assert same(out, eager[i]) and same(between, eager[(i + 1) % 3])


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [257, 264, 513, 520, 776, 1032, 1040, 1049, 1500, 2050, 2064, 3000, 4100, 8193])
def test_rows_that_do_not_fill_the_waves(dtype, V):
    """Waves with few packs or none take none or little of the entries that are looked for."""
    print(f"[top] {dtype} V={V} waves", flush=True)
    rng = np.random.default_rng(V)
    logits = logits_of(rng, (1, 9, V), DTYPES[dtype])
    for k in (1, 17, 64, 65, 130, 256):
        check(logits, k)
