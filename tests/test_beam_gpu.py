"""beam_step and beam_reorder on the device; tolerances in generation_cases.py."""

import numpy as np
import pytest
import torch

import dot_amd
from generation_cases import DTYPES, SUM, array, check_beam, logits_of
from oracle import generation as oracle

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def check(logits, scores, k=None, tau=1.0, finished=None, eos=None, x=None):
    x = logits.to(DEV) if x is None else x
    s = torch.as_tensor(np.asarray(scores, np.float32)).to(DEV)
    f = None if finished is None else torch.as_tensor(finished).to(DEV)
    r = dot_amd.beam_step(x, s, k=k, tau=tau, finished=f, eos=eos)
    check_beam(r, logits, scores, logits.shape[1] if k is None else k, tau, finished, eos)
    return r


def scores_of(rng, B, W):
    return -np.sort(20 + 6 * rng.random((B, W)), 1)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("W", [1, 2, 3, 8, 17, 64, 128])
@pytest.mark.parametrize("V", [2, 9, 255, 2049, 4099])
def test_beams(dtype, W, V):
    print(f"[beam] {dtype} W={W} V={V}", flush=True)
    rng = np.random.default_rng(W * V)
    logits, scores = logits_of(rng, (2, W, V), DTYPES[dtype]), scores_of(rng, 2, W)
    check(logits, scores)
    for k in sorted({1, min(2 * W, W * V, 256), min(256, W * V)}):
        check(logits, scores, k=k, tau=0.7)
    finished = rng.random((2, W)) < 0.4
    check(logits, scores, k=min(2 * W, 256), finished=finished, eos=1)
    check(logits, scores, finished=np.ones((2, W), bool), eos=0)


@pytest.mark.parametrize("B,W,V,k", [(1, 1, 131072, 200), (1, 4, 100003, 8), (3, 5, 50021, 33), (64, 8, 4000, 16),
                                     (2, 16, 160001, 256), (300, 4, 300, 4), (1, 3, 400000, 100)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_sizes(B, W, V, k, dtype):
    print(f"[beam] {dtype} B={B} W={W} V={V} k={k}", flush=True)
    rng = np.random.default_rng(V)
    logits, scores = logits_of(rng, (B, W, V), DTYPES[dtype]), scores_of(rng, B, W)
    finished = rng.random((B, W)) < 0.2
    check(logits, scores, k=k, tau=1.3, finished=finished, eos=2)


def test_closed_beams_and_empty_slots():
    """The first step has one hypothesis; closed and finished rows are not read."""
    rng = np.random.default_rng(1)
    for V in (40, 5000, 70000):
        logits = logits_of(rng, (3, 6, V), torch.float32)
        scores = np.full((3, 6), -np.inf)
        scores[0, 0] = scores[1, 3] = 0.0
        a = check(logits, scores, k=12)
        assert (a.beams[0] == 0).all() and (a.beams[1] == 3).all() and (a.beams[2] == -1).all()
        finished = np.zeros((3, 6), bool)
        finished[0, 1] = finished[0, 2] = True  # closed and finished: has no continuation either
        scores[0, 2] = -5.0
        a = check(logits, scores, k=12, finished=finished, eos=7)
        dirty = logits.clone()
        dirty[torch.as_tensor(~(scores > -np.inf) | finished)] = float("nan")
        s, f = torch.as_tensor(scores.astype(np.float32)).to(DEV), torch.as_tensor(finished).to(DEV)
        b = dot_amd.beam_step(dirty.to(DEV), s, k=12, finished=f, eos=7)
        assert torch.equal(a.scores, b.scores) and torch.equal(a.beams, b.beams) and torch.equal(a.tokens, b.tokens)
        # fewer continuations than asked for
        few = torch.full((3, 6, V), -float("inf"))
        few[0, 0, 5], few[0, 2, 1], few[1, 3, 9] = 1.0, 2.0, 3.0
        r = check(few, scores, k=12, finished=finished, eos=7)
        assert int((r.beams >= 0).sum()) == 3


def test_ties():
    """Equal totals by beam, then by logit, then by token, exactly."""
    for V in (30, 3000):
        rng = np.random.default_rng(V)
        row = np.round(rng.standard_normal(V))
        for W, k in ((5, 5), (5, 20), (64, 128), (128, 256)):
            logits = torch.as_tensor(np.broadcast_to(row, (2, W, V)).astype(np.float32).copy())
            scores = np.zeros((2, W))
            scores[1] = -np.arange(W) // 3
            r = check(logits, scores, k=k)
            _, beams, tokens, _ = oracle.beam_step(array(logits), scores, k)
            assert np.array_equal(r.beams.cpu().numpy(), beams) and np.array_equal(r.tokens.cpu().numpy(), tokens)
    # totals of neighbouring logits that rounding makes equal, the larger logit behind the other in the row
    for V in (600, 40000):
        x = torch.full((1, 3, V), -5.0)
        near = 1.0 + 2.0**-23 * torch.arange(40)
        for w in range(3):
            x[0, w, torch.arange(40) * (V // 40)] = near
            x[0, w, V - 1] = 30.0
        r = dot_amd.beam_step(x.to(DEV), torch.zeros(1, 3, device=DEV), k=100)
        got = [(w, v) for w, v in zip(r.beams[0].tolist(), r.tokens[0].tolist())]
        assert got[:3] == [(0, V - 1), (1, V - 1), (2, V - 1)]
        rest = [(w, v) for s, w, v in sorted(((-float(s), w, i) for i, (s, (w, _)) in enumerate(zip(r.scores[0], got))))[3:]
                for v in [got[v][1]]]
        assert rest == got[3:]
        for w in range(3):  # of one beam by logit, wherever the totals are equal
            mine = [v for u, v in got[3:] if u == w]
            assert mine == sorted(mine, reverse=True)
    # rows that lie at other offsets tie all the same
    V, W = 1001, 7
    flat = torch.zeros(W * (V + 3), dtype=torch.bfloat16, device=DEV)
    x = flat.view(W, V + 3)[:, 1 : V + 1]
    x[:] = torch.as_tensor(np.random.default_rng(0).standard_normal(V).astype(np.float32)).to(DEV)
    r = dot_amd.beam_step(x, torch.full((W,), -3.5, device=DEV))
    assert r.beams.tolist() == list(range(W)) and (r.tokens == r.tokens[0]).all() and (r.scores == r.scores[0]).all()


def test_nan_and_infinite_logits():
    rng = np.random.default_rng(2)
    logits, scores = logits_of(rng, (1, 4, 700), torch.float32), scores_of(rng, 1, 4)
    logits[0, 1, 5] = float("nan")
    logits[0, 2, 5] = float("inf")
    logits[0, 3, 100:] = torch.finfo(torch.float32).min
    r = check(logits, scores, k=50)
    assert set(r.beams[0].tolist()) <= {0, 3}
    scores[0, 0] = np.nan
    r = check(logits, np.where(np.isnan(scores), -np.inf, scores), k=50)
    s = torch.as_tensor(scores.astype(np.float32)).to(DEV)
    assert torch.equal(dot_amd.beam_step(logits.to(DEV), s, k=50).tokens, r.tokens)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_layouts(dtype):
    rng = np.random.default_rng(3)
    logits = logits_of(rng, (4, 6, 520), DTYPES[dtype])
    views = {
        "last position": lambda t: t[:, ::2],
        "offset": lambda t: t[:, :, 3:503],
        "odd rows": lambda t: t[::2, 1::2, 1:],
        "columns": lambda t: t[:, :, ::3],
        "transposed": lambda t: t.transpose(0, 1),
    }
    for name, view in views.items():
        print(f"[beam] {dtype} {name}", flush=True)
        v = view(logits).contiguous()
        check(v, scores_of(rng, v.shape[0], v.shape[1]), x=view(logits.to(DEV)))
    s = torch.as_tensor(scores_of(rng, 4, 6)).to(DEV)
    a = dot_amd.beam_step(logits.to(DEV), s, finished=s < -23, eos=3)
    b = dot_amd.beam_step(logits[2].to(DEV), s.float()[2], finished=s[2] < -23, eos=3)
    assert all(torch.equal(getattr(a, n)[2], getattr(b, n)) for n in ("scores", "beams", "tokens", "finished"))
    st = s.t().contiguous().t()
    c = dot_amd.beam_step(logits.to(DEV), st, finished=st < -23, eos=3)
    assert torch.equal(a.scores, c.scores)
    assert dot_amd.beam_step(torch.zeros(0, 3, 5, device=DEV), torch.zeros(0, 3, device=DEV)).scores.shape == (0, 3)


# ---------------------------------------------------------------------------
# beam_reorder
# ---------------------------------------------------------------------------
TYPES = [torch.bfloat16, torch.float32, torch.int64, torch.uint8, torch.int16, torch.complex128]


def state_of(gen, shape, dtype):
    n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 255, (max(n, 1),), dtype=torch.uint8, device=DEV, generator=gen)[:n]
    return raw.view(dtype).view(shape) if n else torch.empty(shape, dtype=dtype, device=DEV)


def bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy() if t.numel() else np.zeros(0, np.uint8)


def reorder_plain(state, beams, lengths=None, dim=None):
    new = state.clone()
    dim = dim + state.dim() if dim is not None and dim < 0 else dim
    for b, parents in enumerate(beams.tolist()):
        for w, p in enumerate(parents):
            if not 0 <= p < len(parents):
                continue
            old, into = state[b, p], new[b, w]
            if lengths is not None:
                used = min(max(int(lengths[b]), 0), old.shape[dim - 2])
                old, into = old.narrow(dim - 2, 0, used), into.narrow(dim - 2, 0, used)
            into.copy_(old)
    return new


def check_reorder(states, beams, lengths=None, dim=None, guards=()):
    want = [reorder_plain(t, beams, lengths, dim) for t in states]
    before = [g.clone() for g in guards]
    dot_amd.beam_reorder(states, beams, lengths=lengths, dim=dim)
    for t, w in zip(states, want):
        assert np.array_equal(bits(t), bits(w))
    for g, was in zip(guards, before):
        assert np.array_equal(bits(g), bits(was))  # NaN among them


def parents(rng, B, W, kind, dtype=torch.int32):
    p = {"random": rng.integers(0, W, (B, W)), "same": np.broadcast_to(np.arange(W), (B, W)),
         "rotated": np.broadcast_to(np.roll(np.arange(W), 1), (B, W)), "one": np.full((B, W), W - 1),
         "outside": rng.integers(-2, W + 2, (B, W))}[kind]
    return torch.as_tensor(np.ascontiguousarray(p), dtype=dtype).to(DEV)


@pytest.mark.parametrize("kind", ["random", "same", "rotated", "one", "outside"])
@pytest.mark.parametrize("W", [1, 2, 4, 5, 8, 16, 17, 32, 33, 128])
def test_parents(kind, W):
    """Every type in one call: units of 16 bytes to 1, each group of beams."""
    print(f"[reorder] {kind} W={W}", flush=True)
    rng, gen = np.random.default_rng(W), torch.Generator(DEV).manual_seed(W)
    beams = parents(rng, 3, W, kind, torch.int64 if W % 2 else torch.int32)
    states = [state_of(gen, (3, W, 5, n), t) for t in TYPES for n in (1, 3, 8, 37)]
    check_reorder(states, beams)
    lengths = torch.as_tensor([0, 3, 9], device=DEV)
    check_reorder(states, beams, lengths, 2)
    check_reorder([state_of(gen, (3, W), torch.float32)], beams)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8, torch.int64])
def test_cache_layouts(dtype):
    """Heads before positions, positions before heads, positions innermost or outermost, views, odd sizes."""
    rng, gen = np.random.default_rng(1), torch.Generator(DEV).manual_seed(1)
    B, W, H, S, D = 2, 4, 3, 21, 10
    beams = parents(rng, B, W, "random")
    lengths = torch.as_tensor([5, 20], dtype=torch.int32, device=DEV)
    heads = state_of(gen, (B, W, H, S, D), dtype)
    check_reorder([heads], beams, lengths, 3)
    check_reorder([heads], beams, lengths, -2)
    check_reorder([heads.transpose(3, 4)], beams, lengths, 4)
    check_reorder([state_of(gen, (B, W, S, H, D), dtype)], beams, lengths, 2)
    check_reorder([state_of(gen, (S, B, W, H, D), dtype).permute(1, 2, 0, 3, 4)], beams, lengths, 2)
    check_reorder([state_of(gen, (W, B, H, S, D), dtype).transpose(0, 1)], beams, lengths, 3)
    check_reorder([state_of(gen, (B * W, H, S, D), dtype).unflatten(0, (B, W))], beams, lengths, 3)
    # a slice of a longer cache: what lies behind is left alone
    long = state_of(gen, (B, W, H, S + 9, D), dtype)
    rest = long[:, :, :, S:]
    check_reorder([long[:, :, :, :S]], beams, lengths, 3, guards=[rest])
    check_reorder([long[:, :, :, :S]], beams, guards=[rest])
    # keys and values of one tensor, apart and interleaved
    both = state_of(gen, (2, B, W, H, S, D), dtype)
    check_reorder([both[0], both[1]], beams, lengths, 3)
    both = state_of(gen, (B, W, 2, H, S, D), dtype)
    check_reorder([both[:, :, 0], both[:, :, 1]], beams, lengths, 3)
    # unaligned
    raw = state_of(gen, (B * W * S * D + 5,), dtype)
    check_reorder([raw[3 : 3 + B * W * S * D].view(B, W, S, D)], beams, lengths, 2, guards=[raw[:3], raw[-2:]])


def test_many_states():
    rng, gen = np.random.default_rng(2), torch.Generator(DEV).manual_seed(2)
    beams = parents(rng, 3, 6, "random")
    states = [state_of(gen, (3, 6, 1 + i % 5, 17 + i), TYPES[i % 6]) for i in range(75)]
    check_reorder(states, beams)
    dot_amd.beam_reorder(states[0], beams)
    dot_amd.beam_reorder([], beams)
    dot_amd.beam_reorder([torch.zeros(3, 6, 0, device=DEV)], beams)
    dot_amd.beam_reorder([torch.zeros(0, 6, 2, device=DEV)], torch.zeros(0, 6, dtype=torch.int32, device=DEV))


def test_large_offsets():
    """Beams beyond 2^32 bytes of each other."""
    B, W = 2, 3
    state = torch.empty(B, W, 1 << 30, dtype=torch.int16, device=DEV)
    for b in range(B):
        for w in range(W):
            state[b, w].fill_(10 * b + w)
            state[b, w, -1] = 1000 + 10 * b + w
    dot_amd.beam_reorder([state], torch.tensor([[2, 0, 0], [1, 1, 0]], dtype=torch.int32, device=DEV))
    for b, ps in enumerate([[2, 0, 0], [1, 1, 0]]):
        for w, p in enumerate(ps):
            assert int(state[b, w, -1]) == 1000 + 10 * b + p
            assert bool((state[b, w, :-1] == 10 * b + p).all())


def test_refusals_on_the_device():
    t = torch.zeros(2, 4, 6, device=DEV)
    beams = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
    for states in ([t, t], [t, t[:, :, :3]], [t[:, :1].expand(2, 4, 6)], [t[:1].expand(2, 4, 6)],
                   [t.view(-1).as_strided((2, 4, 6), (20, 4, 1))]):
        with pytest.raises(ValueError, match="share memory|overlap"):
            dot_amd.beam_reorder(states, beams)
    with pytest.raises(ValueError, match="share memory"):
        dot_amd.beam_reorder([beams], beams)
    with pytest.raises(ValueError, match="on cuda"):
        dot_amd.beam_reorder([t.cpu()], beams)
    with pytest.raises(ValueError, match="separate dimensions"):
        dot_amd.beam_reorder([torch.zeros(2, 4, 3, 4, 5, 6, device=DEV)[:, :, ::2, ::2, ::2, ::2]], beams)
    assert (t == 0).all()


def test_kept_states_are_noticed():
    """What autograd keeps of a state that is reordered afterwards is not used unnoticed."""
    w = torch.ones(2, 4, 6, device=DEV, requires_grad=True)
    t = torch.rand(2, 4, 6, device=DEV)
    out = (w * t).sum()
    dot_amd.beam_reorder([t], torch.zeros(2, 4, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()
    with pytest.raises(ValueError, match="require a gradient"):
        dot_amd.beam_reorder([w], torch.zeros(2, 4, dtype=torch.int32, device=DEV))
    with torch.no_grad():
        dot_amd.beam_reorder([w], torch.zeros(2, 4, dtype=torch.int32, device=DEV))


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
class Bigram:
    """A language model of a state that a step adds the token's vector to: what beams hold has to follow them."""

    def __init__(self, V, D, dev, seed=0):
        rng = np.random.default_rng(seed)
        make = lambda *s: torch.as_tensor(rng.standard_normal(s).astype(np.float32)).to(dev)  # noqa: E731
        self.vectors, self.out = make(V, D), make(D, V)

    def logits(self, state):
        return torch.tanh(state) @ self.out

    def answers(self, tokens):
        """Logits of each position of (..., S) tokens."""
        v = self.vectors[tokens]
        return self.logits(torch.cumsum(v, -2) - v)


def search(model, B, W, S, eos, V, D, dev):
    state = torch.zeros(B, W, D, device=dev)
    tokens = torch.full((B, W, S), eos, device=dev)
    scores = torch.full((B, W), -float("inf"), device=dev)
    scores[:, 0] = 0
    finished = torch.zeros(B, W, dtype=torch.bool, device=dev)
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)
    for s in range(S):
        r = dot_amd.beam_step(model.logits(state), scores, finished=finished, eos=eos)
        dot_amd.beam_reorder([state], r.beams)
        dot_amd.beam_reorder(tokens, r.beams, lengths=lengths, dim=2)
        tokens[:, :, s] = r.tokens
        state += model.vectors[r.tokens.long()]
        scores, finished = r.scores, r.finished
        lengths += 1
    return tokens, scores, finished


def test_search_scores_and_losses(dev="cuda"):
    """A search's scores are the log-probabilities of its hypotheses, which a student is then taught by."""
    B, W, S, V, D, eos = 3, 5, 7, 60, 8, 4
    model, student = Bigram(V, D, dev), Bigram(V, D, dev, seed=1)
    tokens, scores, finished = search(model, B, W, S, eos, V, D, dev)
    ended = (tokens == eos).cumsum(-1)
    answer = (ended == 0) | ((ended == 1) & (tokens == eos))   # up to the first eos
    logits = model.answers(tokens).flatten(0, 1)
    total = dot_amd.sequence_logp(logits, tokens.flatten(0, 1), mask=answer.flatten(0, 1))
    # S steps, each to 4e-6 as sequence_logp's own, and half a step of fp32 of a sum
    bound = S * (2 * 4e-6 + 2.0**-24 * float(scores.abs().max()))
    assert float((total.view(B, W) - scores).abs().max()) <= bound
    assert torch.equal(finished, (tokens == eos).any(-1))
    assert (scores[:, 1:] <= scores[:, :-1]).all()
    for b in range(B):
        assert len({tuple(t) for t in tokens[b].tolist()}) == W
    # the best one is what an exhaustive search of two steps finds
    two, best, _ = search(model, 1, V, 2, eos, V, D, dev)
    first = torch.log_softmax(model.logits(torch.zeros(D, device=dev)), -1)
    second = torch.log_softmax(model.logits(model.vectors), -1)
    all_ = first[:, None] + second
    all_[eos] = -float("inf")
    all_[eos, eos] = first[eos]
    assert abs(float(best[0, 0]) - float(all_.max())) < 1e-5

    # distillation on these answers, and a preference of the best over the others
    teacher = dot_amd.top_logp(logits, 16)
    leaf = student.out.clone().requires_grad_()
    student.out = leaf
    out = student.answers(tokens).flatten(0, 1)
    mask = answer.flatten(0, 1)
    loss = dot_amd.distill_loss(out, teacher.logp, teacher.tokens, mask=mask)
    ratio = dot_amd.sequence_logp(out, tokens.flatten(0, 1), ref_logp=total.detach(), mask=mask).view(B, W)
    plan = torch.full((1, W - 1), 1.0 / (W - 1), device=dev)
    prefer = torch.cat([dot_amd.preference_loss(ratio[b], plan=plan) for b in range(B)])
    (g,) = torch.autograd.grad(loss.mean() + prefer.mean(), leaf)
    # a step against the gradient lowers the sum by its square's length: to a tenth at this size
    with torch.no_grad():
        size = 1e-3 / float(g.norm())
        student.out = leaf - size * g
        out2 = student.answers(tokens).flatten(0, 1)
        loss2 = dot_amd.distill_loss(out2, teacher.logp, teacher.tokens, mask=mask)
        ratio2 = dot_amd.sequence_logp(out2, tokens.flatten(0, 1), ref_logp=total, mask=mask).view(B, W)
        prefer2 = torch.cat([dot_amd.preference_loss(ratio2[b], plan=plan) for b in range(B)])
        student.out = leaf + size * g
        out3 = student.answers(tokens).flatten(0, 1)
        loss3 = dot_amd.distill_loss(out3, teacher.logp, teacher.tokens, mask=mask)
        ratio3 = dot_amd.sequence_logp(out3, tokens.flatten(0, 1), ref_logp=total, mask=mask).view(B, W)
        prefer3 = torch.cat([dot_amd.preference_loss(ratio3[b], plan=plan) for b in range(B)])
    change = float((loss3.mean() + prefer3.mean()).double() - (loss2.mean() + prefer2.mean()).double())
    assert abs(change - 2 * size * float(g.double().square().sum())) <= 0.1 * abs(change)


def test_search_in_a_graph():
    """A step captured once and replayed, with the program's own work between, goes as the eager one."""
    B, W, S, V, D, eos = 2, 4, 6, 500, 8, 3
    model = Bigram(V, D, DEV)
    want = search(model, B, W, S, eos, V, D, DEV)
    state, tokens = torch.zeros(B, W, D, device=DEV), torch.full((B, W, S), eos, device=DEV)
    scores = torch.full((B, W), -float("inf"), device=DEV)
    scores[:, 0] = 0
    finished = torch.zeros(B, W, dtype=torch.bool, device=DEV)
    at = torch.zeros((), dtype=torch.int64, device=DEV)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)

    def step():
        r = dot_amd.beam_step(model.logits(state), scores, finished=finished, eos=eos)
        dot_amd.beam_reorder([state], r.beams)
        dot_amd.beam_reorder([tokens], r.beams, lengths=lengths, dim=2)
        tokens.scatter_(2, at.expand(B, W, 1), r.tokens.long().unsqueeze(2))
        state.add_(model.vectors[r.tokens.long()])
        scores.copy_(r.scores)
        finished.copy_(r.finished)
        at.add_(1)
        lengths.add_(1)

    begin = [t.clone() for t in (state, tokens, scores, finished, at, lengths)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(2):
        for t, v in zip((state, tokens, scores, finished, at, lengths), begin):
            t.copy_(v)
        for _ in range(S):
            graph.replay()
            torch.cuda.synchronize()
            search(model, B, W, 2, eos, V, D, DEV)
        for got, w in zip((tokens, scores, finished), want):
            assert torch.equal(got, w)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("W,k,ahead", [(64, 256, 8), (64, 128, 4), (64, 64, 9), (128, 256, 12), (128, 200, 6), (7, 256, 5)])
def test_beams_that_are_far_ahead(dtype, W, k, ahead):
    """All entries are from the depth of a few beams' lists; with 8 and 12 of 256 entries
    each, more of them than a join ranks."""
    print(f"[beam] {dtype} W={W} k={k} ahead={ahead}", flush=True)
    rng = np.random.default_rng(W * k)
    for V in (1501, 9000):
        logits = logits_of(rng, (2, W, V), DTYPES[dtype])
        scores = scores_of(rng, 2, W)
        scores[0, :ahead] += 50.0
        scores[1, rng.permutation(W)[:ahead]] += 50.0
        check(logits, scores, k=k)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [516, 520, 1032, 1040, 1096, 2050, 2056, 2064, 2120, 3080, 4104])
def test_spans_that_do_not_fill_the_waves(dtype, V):
    print(f"[beam] {dtype} V={V} waves", flush=True)
    rng = np.random.default_rng(V)
    for W in (1, 4, 16):
        logits, scores = logits_of(rng, (1, W, V), DTYPES[dtype]), scores_of(rng, 1, W)
        for k in sorted({1, W, 2 * W + 1, 70, 256}):
            check(logits, scores, k=k)


@pytest.mark.parametrize("W", [48, 63, 64, 65])
def test_parents_of_many_beams(W):
    print(f"[reorder] W={W}", flush=True)
    rng, gen = np.random.default_rng(W), torch.Generator(DEV).manual_seed(W)
    beams = parents(rng, 2, W, "random")
    check_reorder([state_of(gen, (2, W, 7, n), t) for t in TYPES for n in (1, 4, 40)], beams)
    check_reorder([state_of(gen, (2, W, 3, 33, 16), torch.bfloat16)], beams,
                  torch.as_tensor([33, 10], device=DEV), 3)
