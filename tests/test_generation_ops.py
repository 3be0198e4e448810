"""Top log-probabilities, distillation and beam search on the CPU against the float64
definitions, the definitions against differences, and what is refused."""

import ctypes
import importlib
import os

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fw

import dot
import dot_amd
from conftest import ROOT
from generation_cases import DTYPES, check_beam, check_distill, check_top, logits_of, teacher_of
from oracle import generation as oracle

FORMS = [("forward", "bucket"), ("forward", "none"), ("reverse", "bucket")]


# ---------------------------------------------------------------------------
# The definition
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("direction,rest", FORMS)
@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
def test_gradient_by_differences(direction, rest, reduction):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 3, 7))
    logp, tokens = teacher_of(rng, torch.as_tensor(x), 3, tau=0.8)
    tokens[0, 1, 2] = tokens[0, 1, 0]
    tokens[1, 2] = -1
    mask = np.ones((2, 3), bool)
    mask[1, 0] = False
    up = rng.standard_normal((2, 3) if reduction == "none" else 2)
    f = lambda x: (oracle.distill(x, logp, tokens, mask, 0.8, direction, rest, reduction)[0] * up).sum()  # noqa: E731
    _, parts = oracle.distill(x, logp, tokens, mask, 0.8, direction, rest, reduction)
    g = oracle.distill_grad(x.shape, parts, up, 0.8)
    for at in np.ndindex(*x.shape):
        d = np.zeros_like(x)
        d[at] = 1e-5
        # of a central difference: h^2 / 6 of a third derivative of order 1, and 1e-16 / h
        assert abs((f(x + d) - f(x - d)) / 2e-5 - g[at]) < 1e-8


def test_definition_of_whole_distributions():
    """A teacher that names every token: the divergences of two softmaxes."""
    rng = np.random.default_rng(1)
    x, y = rng.standard_normal((1, 1, 6)), rng.standard_normal((1, 1, 6))
    p, q = oracle.log_softmax(y)[0, 0], oracle.log_softmax(x)[0, 0]
    tokens = np.arange(6)[None, None]
    for rest in ("bucket", "none"):
        v, _ = oracle.distill(x, p[None, None], tokens, rest=rest)
        assert abs(v[0] - (np.exp(p) * (p - q)).sum()) < 1e-6  # the teacher's own fp32
    v, _ = oracle.distill(x, p[None, None], tokens, direction="reverse")
    assert abs(v[0] - (np.exp(q) * (q - p)).sum()) < 1e-6


# ---------------------------------------------------------------------------
# CPU tensors
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("V", [1, 2, 9, 300])
def test_cpu_top_logp(dtype, V):
    rng = np.random.default_rng(V)
    logits = logits_of(rng, (2, 4, V), DTYPES[dtype])
    if V > 2:
        logits[0, 0, 1:] = -float("inf")
        logits[0, 1] = -float("inf")
        logits[1, 1, 2] = float("nan")
        logits[1, 2] = 0.5
    mask = np.ones((2, 4), bool)
    mask[1, 3] = False
    for k in {1, min(V, 7), min(V, 256)}:
        check_top(dot_amd.top_logp(logits, k, tau=1.5, mask=torch.as_tensor(mask)), logits, k, 1.5, mask)
    one = dot_amd.top_logp(logits[1], 1)
    assert torch.equal(one.tokens, dot_amd.top_logp(logits, 1).tokens[1])
    wide = torch.zeros(2, 4, 2 * V, dtype=logits.dtype)[..., ::2].copy_(logits)
    assert torch.equal(dot_amd.top_logp(wide, 1).tokens, dot_amd.top_logp(logits, 1).tokens)


@pytest.mark.parametrize("direction,rest", FORMS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("reduction", ["sum", "mean", "none"])
def test_cpu_distill(dtype, direction, rest, reduction):
    rng = np.random.default_rng(2)
    logits = logits_of(rng, (3, 5, 40), DTYPES[dtype])
    logp, tokens = teacher_of(rng, logits, 6, tau=0.7)
    tokens[0, 0, 3], tokens[0, 1, 0], tokens[0, 2, 4] = -100, 40, tokens[0, 2, 1]
    logp[0, 3, 2:] = -np.inf
    tokens[0, 4] = -1
    mask = rng.random((3, 5)) < 0.7
    mask[1] = False
    logits[2, 0, tokens[2, 0, 0]] = -float("inf")
    logits[2, 1] = torch.finfo(logits.dtype).min
    lp, tk = torch.as_tensor(logp), torch.as_tensor(tokens)

    def call(x, mask, **kw):
        return dot_amd.distill_loss(x, lp, tk, mask=None if mask is None else torch.as_tensor(mask), **kw)

    kw = dict(tau=0.7, direction=direction, rest=rest, reduction=reduction)
    check_distill(call, logits, logp, tokens, mask=mask, **kw)
    check_distill(call, logits, logp, tokens, **kw)
    one = dot_amd.distill_loss(logits[0], lp[0], tk[0], **kw)
    assert torch.equal(one, call(logits, None, **kw)[0])


def test_cpu_distill_whole_vocabulary():
    """A teacher that names every token leaves nothing but rounding, which is not held against the student."""
    rng = np.random.default_rng(3)
    logits = logits_of(rng, (1, 4, 9), torch.float32)
    logp, tokens = teacher_of(rng, logits, 9)
    lp, tk = torch.as_tensor(logp), torch.as_tensor(tokens)
    for direction, rest in FORMS:
        x = logits.clone().requires_grad_()
        out = dot_amd.distill_loss(x, lp, tk, direction=direction, rest=rest)
        (g,) = torch.autograd.grad(out.sum(), x)
        assert torch.isfinite(out).all() and torch.isfinite(g).all() and float(out) > 0


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_cpu_beam_step(dtype):
    rng = np.random.default_rng(4)
    for W, V in ((1, 5), (4, 30), (9, 300)):
        logits = logits_of(rng, (3, W, V), DTYPES[dtype])
        logits[0, 0, 2] = -float("inf")
        logits[1, 0, 1] = float("nan")
        scores = -np.sort(5 * rng.random((3, W)), 1)
        scores[2, W // 2] = -np.inf
        s, finished = torch.as_tensor(scores.astype(np.float32)), rng.random((3, W)) < 0.4
        for k in (None, 1, min(2 * W, W * V)):
            check_beam(dot_amd.beam_step(logits, s, k=k), logits, scores, k or W)
            r = dot_amd.beam_step(logits, s.double(), k=k, tau=0.6, finished=torch.as_tensor(finished), eos=2)
            check_beam(r, logits, scores, k or W, 0.6, finished, 2)
    ties = torch.zeros(1, 3, 4)
    r = dot_amd.beam_step(ties, torch.zeros(1, 3), k=6)
    assert r.beams.tolist() == [[0, 0, 0, 0, 1, 1]] and r.tokens.tolist() == [[0, 1, 2, 3, 0, 1]]
    one = dot_amd.beam_step(ties[0], torch.zeros(3), k=6, eos=1)
    assert one.beams.tolist() == r.beams[0].tolist() and one.finished.tolist() == [False, True, False, False, False, True]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int64, torch.uint8])
def test_cpu_beam_reorder(dtype):
    rng = np.random.default_rng(5)
    make = lambda *s: torch.as_tensor(rng.integers(0, 100, s)).to(dtype)  # noqa: E731
    B, W, H, S, D = 2, 4, 3, 6, 5
    beams = torch.as_tensor([[3, 0, 0, 7], [-1, 2, 1, 3]])
    lengths = torch.as_tensor([2, 9], dtype=torch.int32)
    as_numbers = lambda t: t.double().numpy()  # noqa: E731
    both = make(B, W, 2, H, S, D)
    layouts = [(make(B, W, H, S, D), 3), (make(B, W, S, H, D), 2), (make(B, W, H, D, S), 4), (make(B, W, S), 2),
               (make(S, B, W, H, D).permute(1, 2, 0, 3, 4), 2), (make(B, W, H, S + 3, D)[:, :, :, :S], 3),
               (both[:, :, 0], 3), (both[:, :, 1], 3)]
    for t, dim in layouts:
        want = oracle.beam_reorder(as_numbers(t), beams.tolist(), lengths.tolist(), dim)
        dot_amd.beam_reorder(t, beams, lengths=lengths, dim=dim)
        assert np.array_equal(as_numbers(t), want)
    states = [t for t, _ in layouts]
    want = [oracle.beam_reorder(as_numbers(t), beams.tolist()) for t in states]
    dot_amd.beam_reorder(states, beams.int())
    assert all(np.array_equal(as_numbers(t), w) for t, w in zip(states, want))
    dot_amd.beam_reorder([make(B, W)], beams)
    dot_amd.beam_reorder([], beams)


@pytest.mark.parametrize("tau", [0.7, 1.0, 1.3])
def test_cpu_logits_are_scaled_in_fp32(tau):
    """As on the device: what beams are compared by."""
    rng = np.random.default_rng(6)
    x = np.full((300, 5), -np.inf, np.float32)
    x[:, 0] = 100.0
    x[:, 4] = 40 + 5 * rng.random(300)
    inv = np.float32(1) / np.float32(tau)
    r = dot_amd.top_logp(torch.as_tensor(x), 2, tau=tau)
    assert np.array_equal(r.logp[:, 1].numpy(), x[:, 4] * inv - x[:, 0] * inv)
    s = dot_amd.beam_step(torch.as_tensor(x[:, None]), torch.full((300, 1), -2.0), k=2, tau=tau)
    want = (-2.0 + (x[:, 4] * inv - x[:, 0] * inv).astype(np.float64)).astype(np.float32)
    assert np.array_equal(s.scores[:, 1].numpy(), want)


def test_inference_states():
    with torch.inference_mode():
        t = torch.arange(8.0).view(1, 2, 4)
        dot_amd.beam_reorder(t, torch.tensor([[1, 1]]))
    assert t.tolist() == [[[4, 5, 6, 7], [4, 5, 6, 7]]]
    with pytest.raises(ValueError, match="inference"):
        dot_amd.beam_reorder(t, torch.tensor([[1, 0]]))


def test_cpu_search_scores_and_losses():
    import test_beam_gpu

    test_beam_gpu.test_search_scores_and_losses("cpu")


def test_cpu_empty():
    assert dot_amd.top_logp(torch.zeros(2, 0, 4), 2).tokens.shape == (2, 0, 2)
    lp, tk = torch.zeros(2, 0, 3), torch.zeros(2, 0, 3, dtype=torch.int32)
    assert dot_amd.distill_loss(torch.zeros(2, 0, 4), lp, tk).tolist() == [0, 0]
    assert dot_amd.beam_step(torch.zeros(0, 2, 4), torch.zeros(0, 2)).beams.shape == (0, 2)


# ---------------------------------------------------------------------------
# Names, derivatives, refusals
# ---------------------------------------------------------------------------
def test_modules_and_names():
    rng = np.random.default_rng(6)
    x = logits_of(rng, (2, 3, 20), torch.float32)
    a, b = dot.TopLogp(4, tau=0.5)(x), dot.top_logp(x, 4, tau=0.5)
    assert torch.equal(a.logp, b.logp) and isinstance(a, dot.TopLogpResult)
    loss = dot.DistillLoss(0.5, "reverse", "bucket", "sum")(x, a.logp, a.tokens)
    assert torch.equal(loss, dot.distill_loss(x, a.logp, a.tokens, tau=0.5, direction="reverse", reduction="sum"))
    assert isinstance(dot.beam_step(x, torch.zeros(2, 3)), dot.BeamResult)
    assert importlib.import_module("dot.distillation").distill_loss is dot_amd.distill_loss
    assert importlib.import_module("dot.beam").beam_step is dot_amd.beam_step


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_derivatives(dev):
    """Once, backwards, by the student's logits: anything else is refused, or a constant."""
    rng = np.random.default_rng(7)
    x = logits_of(rng, (2, 3, 20), torch.float32).to(dev)
    t = dot_amd.top_logp(x.clone().requires_grad_(), 5)
    assert not t.logp.requires_grad
    f = lambda x: dot_amd.distill_loss(x, t.logp, t.tokens)  # noqa: E731
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(fw.make_dual(x, torch.ones_like(x)))
        constant = dot_amd.distill_loss(x, fw.make_dual(t.logp, torch.ones_like(t.logp)), t.tokens)
        assert fw.unpack_dual(constant).tangent is None
        assert fw.unpack_dual(dot_amd.top_logp(fw.make_dual(x, torch.ones_like(x)), 2).logp).tangent is None
        r = dot_amd.beam_step(fw.make_dual(x, torch.ones_like(x)), torch.zeros(2, 3, device=dev))
        assert fw.unpack_dual(r.scores).tangent is None
    x.requires_grad_()
    assert not dot_amd.beam_step(x, torch.zeros(2, 3, device=dev, requires_grad=True)).scores.requires_grad
    out = f(x)
    (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
    for total in (g.sum(), out.sum() + (g**2).sum()):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(total, x, retain_graph=True)
    up = torch.ones_like(out).requires_grad_()
    (g,) = torch.autograd.grad(out, x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(g.sum(), up)
    with torch.no_grad():
        assert not f(x).requires_grad


def test_refusals():
    x, lp, tk = torch.zeros(2, 5, 8), torch.zeros(2, 5, 3), torch.zeros(2, 5, 3, dtype=torch.int32)
    s, t, b = torch.zeros(2, 5), torch.zeros(2, 5, 4), torch.zeros(2, 5, dtype=torch.int32)
    one = torch.ones(2, 5, dtype=torch.bool)
    bad = [
        (lambda: dot.top_logp(x, 0), "k must be"), (lambda: dot.top_logp(x, 9), "k must be"),
        (lambda: dot.top_logp(x, 2.0), "k must be"), (lambda: dot.top_logp(x, True), "k must be"),
        (lambda: dot.top_logp(torch.zeros(1, 1, 300), 257), "k must be"),
        (lambda: dot.top_logp(x.double(), 2), "float32"), (lambda: dot.top_logp(x[0, 0], 2), "shape"),
        (lambda: dot.top_logp(torch.zeros(1, 2, 0), 1), "V >= 1"), (lambda: dot.top_logp(x, 2, tau=0.0), "tau"),
        (lambda: dot.top_logp(x, 2, tau=float("inf")), "tau"), (lambda: dot.top_logp(x, 2, mask=torch.ones(2, 5)), "mask"),
        (lambda: dot.top_logp(x, 2, mask=one[:, :4]), "mask"),
        (lambda: dot.distill_loss(x.double(), lp, tk), "float32"), (lambda: dot.distill_loss(x, lp, tk[:, :4]), "teacher_tokens"),
        (lambda: dot.distill_loss(x, lp, tk.float()), "teacher_tokens"), (lambda: dot.distill_loss(x, lp[..., :2], tk), "teacher_logp"),
        (lambda: dot.distill_loss(x, lp.long(), tk), "teacher_logp"), (lambda: dot.distill_loss(x, lp[..., :0], tk[..., :0]), "tokens of a position"),
        (lambda: dot.distill_loss(x, torch.zeros(2, 5, 257), torch.zeros(2, 5, 257, dtype=torch.int32)), "tokens of a position"),
        (lambda: dot.distill_loss(x, lp, tk, direction="back"), "direction"), (lambda: dot.distill_loss(x, lp, tk, rest="drop"), "rest"),
        (lambda: dot.distill_loss(x, lp, tk, direction="reverse", rest="none"), "bucket"),
        (lambda: dot.distill_loss(x, lp, tk, reduction="max"), "reduction"), (lambda: dot.distill_loss(x, lp, tk, tau=-1.0), "tau"),
        (lambda: dot.distill_loss(x, lp, tk, mask=one[0]), "mask"),
        (lambda: dot.beam_step(x, s[:, :4]), "scores"), (lambda: dot.beam_step(x, s.long()), "scores"),
        (lambda: dot.beam_step(x.double(), s), "float32"), (lambda: dot.beam_step(x, s, k=0), "k must be"),
        (lambda: dot.beam_step(x, s, k=41), "k must be"), (lambda: dot.beam_step(torch.zeros(1, 2, 300), s[:1, :2], k=257), "k must be"),
        (lambda: dot.beam_step(torch.zeros(1, 129, 3), torch.zeros(1, 129)), "beams"),
        (lambda: dot.beam_step(torch.zeros(1, 0, 3), torch.zeros(1, 0)), "beams"), (lambda: dot.beam_step(x, s, eos=8), "eos"),
        (lambda: dot.beam_step(x, s, eos=-1), "eos"), (lambda: dot.beam_step(x, s, eos=True), "eos"),
        (lambda: dot.beam_step(x, s, finished=one), "needs eos"), (lambda: dot.beam_step(x, s, finished=s, eos=1), "finished"),
        (lambda: dot.beam_step(x, s, finished=one[:1], eos=1), "finished"), (lambda: dot.beam_step(x, s, tau=0.0), "tau"),
        (lambda: dot.beam_reorder(t, b.float()), "beams"), (lambda: dot.beam_reorder(t, b[0]), "beams"),
        (lambda: dot.beam_reorder(t, torch.zeros(2, 129, dtype=torch.int32)), "beams are supported"),
        (lambda: dot.beam_reorder(t[:1], b), "states must"), (lambda: dot.beam_reorder(t[0], b), "states must"),
        (lambda: dot.beam_reorder(t, b, lengths=b[:, 0]), "needs dim"),
        (lambda: dot.beam_reorder(t, b, lengths=b[:1, 0], dim=2), "lengths"), (lambda: dot.beam_reorder(t, b, lengths=s[:, 0], dim=2), "lengths"),
        (lambda: dot.beam_reorder(t, b, lengths=b[:, 0], dim=1), "dim"), (lambda: dot.beam_reorder(t, b, lengths=b[:, 0], dim=3), "dim"),
        (lambda: dot.beam_reorder(t, b, lengths=b[:, 0], dim=-2), "dim"), (lambda: dot.beam_reorder(t, b, lengths=b[:, 0], dim=True), "dim"),
        (lambda: dot.beam_reorder(t.clone().requires_grad_(), b), "gradient"), (lambda: dot.beam_reorder([t, t], b), "share memory"),
        (lambda: dot.beam_reorder([t, t[..., 1:]], b), "share memory"), (lambda: dot.beam_reorder(t[:1].expand(2, 5, 4), b), "overlap"),
        (lambda: dot.beam_reorder(t.view(-1).as_strided((2, 5, 4), (20, 3, 1)), b), "overlap"), (lambda: dot.beam_reorder([b], b), "share memory"),
        (lambda: dot.beam_reorder(torch.zeros(2, 5, 3, 4, 5, 6)[:, :, ::2, ::2, ::2, ::2], b), "separate dimensions"),
    ]
    for i, (f, text) in enumerate(bad):
        with pytest.raises(ValueError, match=text):
            f()
            pytest.fail(f"call {i} ({text}) was not refused")


@pytest.mark.gpu
def test_limits_of_the_device_are_refused_as_values():
    dev = torch.device("cuda", 0)
    x = torch.zeros(1, 2, 4)
    lp, tk = torch.zeros(1, 2, 1), torch.zeros(1, 2, 1, dtype=torch.int32)
    for tau in (1e-21, 1e21):
        dot_amd.top_logp(x, 1, tau=tau)
        for f in (lambda: dot_amd.top_logp(x.to(dev), 1, tau=tau), lambda: dot_amd.beam_step(x.to(dev), torch.zeros(1, 2, device=dev), tau=tau),
                  lambda: dot_amd.distill_loss(x.to(dev), lp.to(dev), tk.to(dev), tau=tau)):
            with pytest.raises(ValueError, match="tau"):
                f()
    few = torch.zeros(1, 1, 1, device=dev)
    for shape in ((1, 2**23 + 1, 1), (1, 2**22 + 1, 2**18 + 1)):
        with pytest.raises(ValueError, match="positions"):
            dot_amd.top_logp(few.expand(shape), 1)
    with pytest.raises(ValueError, match="vocabulary"):
        dot_amd.top_logp(few.expand(1, 1, 2**24 + 1), 1)
    with pytest.raises(RuntimeError, match="must be on"):
        dot_amd.distill_loss(x.to(dev), lp, tk)


# ---------------------------------------------------------------------------
# C ABI: bad arguments are refused on the host
# ---------------------------------------------------------------------------
P, I, I64, D, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t


def struct(*fields):
    return type("Args", (ctypes.Structure,), {"_fields_": list(fields)})


Top = struct(("logits", P), ("dtype", I), ("sb", I64), ("ss", I64), ("B", I), ("S", I), ("V", I), ("k", I), ("mask", P),
             ("tau", D), ("logp", P), ("tokens", P), ("workspace", P), ("workspace_bytes", Z))
Fwd = struct(("logits", P), ("dtype", I), ("sb", I64), ("ss", I64), ("B", I), ("S", I), ("V", I), ("K", I), ("tokens", P),
             ("tokens64", I), ("logp", P), ("mask", P), ("tau", D), ("direction", I), ("rest", I), ("reduction", I),
             ("out", P), ("row_stats", P), ("own_tokens", P), ("own_grad", P), ("weight", P), ("workspace", P),
             ("workspace_bytes", Z))
Bwd = struct(("logits", P), ("dtype", I), ("sb", I64), ("ss", I64), ("B", I), ("S", I), ("V", I), ("K", I), ("tau", D),
             ("reduction", I), ("mask", P), ("row_stats", P), ("own_tokens", P), ("own_grad", P), ("weight", P),
             ("grad_out", P), ("grad_out_scalar", I), ("grad_logits", P))
Step = struct(("logits", P), ("dtype", I), ("sb", I64), ("sw", I64), ("B", I), ("W", I), ("V", I), ("n", I), ("tau", D),
              ("scores", P), ("finished", P), ("eos", I), ("out_scores", P), ("out_beams", P), ("out_tokens", P),
              ("out_finished", P), ("workspace", P), ("workspace_bytes", Z))
State = struct(("data", P), ("sb", I64), ("sw", I64), ("so", I64), ("sp", I64), ("outer", I64), ("positions", I64),
               ("inner", I64))
Reorder = struct(("states", ctypes.POINTER(State)), ("count", I), ("B", I), ("W", I), ("beams", P), ("beams64", I),
                 ("lengths", P), ("lengths64", I))
INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(os.path.join(ROOT, "dot_amd", "libdot_amd.so"))
    lib.dot_last_error.restype = ctypes.c_char_p
    for name in ("dot_top_logp", "dot_distill_forward", "dot_beam_step"):
        getattr(lib, name + "_workspace_bytes").restype = ctypes.c_size_t
    return lib


def test_c_abi_refusals(lib):
    some = 4096  # an address that is never read: every call here is refused before a launch

    def refused(name, code, text, args):
        args = () if args is None else (ctypes.byref(args),)
        more = () if name.endswith("_check") else (None,)
        assert getattr(lib, name)(*(args or (None,)), *more) == code
        assert text in lib.dot_last_error().decode()

    t = dict(logits=some, B=2, S=3, V=16, k=4, tau=1.0, logp=some, tokens=some)
    f = "dot_top_logp"
    refused(f, INVALID, "NULL", None)
    refused(f, INVALID, "dtype", Top(**{**t, "dtype": 7}))
    refused(f, INVALID, "V must", Top(**{**t, "V": 0}))
    refused(f, INVALID, "k must be at most V", Top(**{**t, "k": 17}))
    refused(f, INVALID, "at least one", Top(**{**t, "k": 0}))
    refused(f, UNSUPPORTED, "DOT_TOP_MAX", Top(**{**t, "V": 1000, "k": 257}))
    refused(f, UNSUPPORTED, "2^24", Top(**{**t, "V": (1 << 24) + 1}))
    refused(f, UNSUPPORTED, "2^23", Top(**{**t, "B": 4096, "S": 4096}))
    refused(f, INVALID, "tau", Top(**{**t, "tau": 0.0}))
    refused(f, UNSUPPORTED, "tau", Top(**{**t, "tau": 1e-30}))
    refused(f, INVALID, "non-NULL", Top(**{**t, "tokens": None}))
    refused(f, INVALID, ">= 0", Top(**{**t, "B": -1}))
    refused(f, WORKSPACE, "workspace", Top(**{**t, "V": 200000}))
    need = lib.dot_top_logp_workspace_bytes(2, 3, 200000, 0, 4)
    assert need > 0 and lib.dot_top_logp_workspace_bytes(-1, 3, 16, 0, 4) == 0
    refused(f, WORKSPACE, "workspace", Top(**{**t, "V": 200000}, workspace=some, workspace_bytes=need - 1))

    s = dict(logits=some, B=2, S=3, V=16, K=4, tokens=some, logp=some, tau=1.0, reduction=1, out=some)
    f = "dot_distill_forward"
    refused(f, INVALID, "K must", Fwd(**{**s, "K": 0}))
    refused(f, UNSUPPORTED, "DOT_TOP_MAX", Fwd(**{**s, "K": 257}))
    refused(f, INVALID, "direction", Fwd(**{**s, "direction": 2}))
    refused(f, INVALID, "rest", Fwd(**{**s, "rest": 2}))
    refused(f, INVALID, "DOT_REST_BUCKET", Fwd(**{**s, "direction": 1, "rest": 1}))
    refused(f, INVALID, "reduction", Fwd(**{**s, "reduction": 5}))
    refused(f, UNSUPPORTED, "2^24", Fwd(**{**s, "V": (1 << 24) + 1}))
    refused(f, UNSUPPORTED, "2^23", Fwd(**{**s, "V": 1 << 24, "B": 1 << 18}))
    refused(f, INVALID, "non-NULL", Fwd(**{**s, "logp": None}))
    refused(f, INVALID, "own_tokens", Fwd(**{**s, "row_stats": some}))
    refused(f, WORKSPACE, "workspace", Fwd(**s))
    b = dict(logits=some, B=2, S=3, V=16, K=4, tau=1.0, reduction=2, row_stats=some, own_tokens=some, own_grad=some,
             grad_out=some, grad_logits=some)
    f = "dot_distill_backward"
    refused(f, INVALID, "weight", Bwd(**b))
    refused(f, INVALID, "non-NULL", Bwd(**{**b, "grad_logits": None}))
    refused(f, INVALID, "tau", Bwd(**{**b, "tau": float("nan")}))

    w = dict(logits=some, B=2, W=3, V=16, n=4, tau=1.0, scores=some, eos=-1, out_scores=some, out_beams=some,
             out_tokens=some)
    f = "dot_beam_step"
    refused(f, INVALID, "W >= 1", Step(**{**w, "W": 0}))
    refused(f, UNSUPPORTED, "DOT_BEAM_MAX", Step(**{**w, "W": 129}))
    refused(f, INVALID, "n must", Step(**{**w, "n": 49}))
    refused(f, UNSUPPORTED, "DOT_TOP_MAX", Step(**{**w, "V": 1000, "n": 257}))
    refused(f, INVALID, "eos", Step(**{**w, "finished": some}))
    refused(f, INVALID, "eos", Step(**{**w, "finished": some, "eos": 16}))
    refused(f, INVALID, "non-NULL", Step(**{**w, "scores": None}))
    refused(f, WORKSPACE, "workspace", Step(**w))
    assert lib.dot_beam_step_workspace_bytes(2, 129, 16, 0, 4) == 0

    def reorder(*states, **kw):
        a = dict(B=2, W=3, beams=1 << 40, count=len(states))
        return Reorder(states=(State * max(1, len(states)))(*states), **{**a, **kw})

    one = dict(data=some, sb=96, sw=32, so=16, sp=4, outer=2, positions=4, inner=4)
    for f in ("dot_beam_reorder", "dot_beam_reorder_check"):
        refused(f, INVALID, "NULL", None)
        refused(f, INVALID, "W >= 1", reorder(State(**one), W=0))
        refused(f, UNSUPPORTED, "DOT_BEAM_MAX", reorder(State(**one), W=129))
        refused(f, INVALID, "non-NULL", reorder(State(**one), beams=None))
        refused(f, INVALID, "non-NULL", reorder(State(**{**one, "data": None})))
        refused(f, INVALID, ">= 0", reorder(State(**{**one, "sw": -32})))
        refused(f, INVALID, "overlap", reorder(State(**{**one, "sw": 31})))
        refused(f, INVALID, "overlap", reorder(State(**{**one, "sb": 90})))
        refused(f, INVALID, "overlap", reorder(State(**{**one, "sp": 0})))
        refused(f, INVALID, "share memory", reorder(State(**one), State(**{**one, "data": some + 188})))
        refused(f, INVALID, "share memory", reorder(State(**one), beams=some + 191))
        refused(f, INVALID, "share memory", reorder(State(**one), lengths=some - 7))
    check = lib.dot_beam_reorder_check
    good = [reorder(State(**one)), reorder(State(**one), State(**{**one, "data": some + 192})), reorder(),
            # interleaved: each in the other's gaps
            reorder(State(**{**one, "sw": 64, "sb": 192}), State(**{**one, "sw": 64, "sb": 192, "data": some + 32})),
            reorder(State(**{**one, "outer": 0, "data": None})), reorder(State(**one), B=0, beams=None)]
    for a in good:
        assert check(ctypes.byref(a)) == 0
