"""The operators on single lattice nodes (transducer_b200.nodes) against their definitions in 64 bits."""
import math

import pytest
import torch

import node_reference as ref
from transducer_b200 import NodeDistillationLoss, TransducerLoss, sample_words, top_words

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -24   # half a step of a 32-bit number


def make(B, T, U, V, N, dtype=torch.float32, seed=0, std=2.0, holes=True, kind="any"):
    g = torch.Generator().manual_seed(seed)
    E = torch.randn(B, T, V, generator=g) * std
    P = torch.randn(B, U, V, generator=g) * std / 2
    raised = torch.randint(0, V, (B, T, 1), generator=g)
    E.scatter_add_(2, raised, 8.0 * torch.rand(B, T, 1, generator=g))
    if kind == "any":
        frames = torch.randint(0, T, (B, N), generator=g)
        positions = torch.randint(0, U, (B, N), generator=g)
    else:   # a way through the lattice
        label = torch.rand(B, N, generator=g) < U / (T + U)
        positions = (label.cumsum(1) - label.long()).clamp(max=U - 1)
        frames = (torch.arange(N) - (label.cumsum(1) - label.long())).clamp(0, T - 1)
    if holes:
        gone = torch.rand(B, N, generator=g) < 0.15
        frames[gone] = -1
    return (E.to(dtype).cuda(), P.to(dtype).cuda(), frames.int().cuda(), positions.int().cuda(), g)


SIZES = [1, 2, 7, 8, 31, 33, 128, 255, 256, 257, 264, 1000, 1023, 1024, 1025, 1032, 4096, 4097, 4104, 10000,
         16384, 16392, 32768, 32769, 40000, 60000, 60001]


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 5, 40, 256])
def test_top_words(V, dtype, k):
    k = min(k, V)
    E, P, frames, positions, _ = make(2, 5, 3, V, 9, dtype, seed=V + k)
    temperature = (1.0, 0.7)[V % 2]
    words, logits, rest = top_words(E, P, frames, positions, k, temperature)
    z, here = ref.scores(E, P, frames, positions)
    w, l, r = ref.top_words(z, here, k, temperature)
    assert torch.equal(words.cpu(), w)
    # the scale and the product are rounded once each
    torch.testing.assert_close(logits.cpu().double(), l, rtol=2 * 2 * UNIT, atol=0.0)
    # the distance to the maximum, its scaling, the exponentials and their sums, the logarithm
    torch.testing.assert_close(rest.cpu().double(), r, rtol=64 * UNIT, atol=128 * UNIT)


@pytest.mark.parametrize("V", [1, 40, 1025, 4096, 12000, 33000, 60000])
@pytest.mark.parametrize("k", [1, 3, 200])
def test_top_words_of_equal_and_masked_scores(V, k):
    k = min(k, V)
    E, P, frames, positions, g = make(3, 4, 2, V, 8, seed=V)
    E[0] = 0.0          # every score the same
    P[0] = -0.0
    E[1] = (E[1] * 0.5).round()       # many equal ones
    P[1] = P[1].round()
    E[2, :, torch.randperm(V, generator=g)[: V - V // 3]] = -math.inf   # fewer than k words left at times
    E[2, 1] = -math.inf
    E[2, 2] = torch.finfo(torch.float32).min
    frames[:, 1], positions[:, 1] = 1, 0
    frames[:, 2], positions[:, 2] = 2, 1
    words, logits, rest = top_words(E, P, frames, positions, k)
    z, here = ref.scores(E, P, frames, positions)
    w, l, r = ref.top_words(z, here, k)
    assert torch.equal(words.cpu(), w)
    assert torch.equal(logits.cpu().double(), l)
    torch.testing.assert_close(rest.cpu().double(), r, rtol=64 * UNIT, atol=128 * UNIT)


@pytest.mark.parametrize("V", [33, 1000, 5000, 60001])
def test_top_words_of_broken_scores(V):
    """NaN stands above everything and +inf above all numbers; the other nodes are what they were."""
    E, P, frames, positions, g = make(2, 4, 2, V, 8, seed=V, holes=False)
    clean = top_words(E, P, frames, positions, 9)
    E[0, 1, V // 3], E[0, 1, V - 1], E[0, 2, 5], E[1, 3, 7] = math.nan, math.nan, math.inf, math.nan
    E[1, 3, 8], E[1, 3, 20] = math.inf, -math.inf
    words, logits, rest = top_words(E, P, frames, positions, 9)
    z, here = ref.scores(E, P, frames, positions)
    w, l, r = ref.top_words(z, here, 9)
    assert torch.equal(words.cpu(), w)
    torch.testing.assert_close(logits.cpu().double(), l, rtol=0, atol=0, equal_nan=True)
    whole = z.isfinite().all(-1)
    torch.testing.assert_close(rest.cpu().double()[whole], r[whole], rtol=64 * UNIT, atol=128 * UNIT)
    assert torch.equal(rest[whole.cuda()], clean[2][whole.cuda()])


def check_sample(E, P, frames, positions, uniforms, **rule):
    words, log_probs = sample_words(E, P, frames, positions, uniforms, **rule)
    z, here = ref.scores(E, P, frames, positions)
    w, l = ref.sample_words(z, here, uniforms, **rule)
    assert torch.equal(words.cpu(), w), (words.cpu() != w).sum()
    # exponentials and their sums in 32 bits or more
    torch.testing.assert_close(log_probs.cpu().double(), l, rtol=4 * UNIT, atol=64 * UNIT, equal_nan=True)
    return words


RULES = [dict(), dict(temperature=0.0), dict(temperature=0.6, top_k=3), dict(top_k=40, top_p=0.8),
         dict(temperature=1.7, top_p=0.95), dict(min_p=0.05), dict(top_p=0.3, min_p=0.2, top_k=7),
         dict(temperature=3.0, top_p=0.999), dict(top_k=700, top_p=0.99, temperature=2.0), dict(min_p=1.0)]


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_words(V, dtype):
    E, P, frames, positions, g = make(2, 6, 4, V, 24, dtype, seed=V + 1, std=1.5)
    uniforms = torch.rand(2, 24, generator=g).cuda()
    uniforms[0, 0], uniforms[0, 1] = 0.0, 1.0 - 2.0 ** -24
    for rule in RULES:
        check_sample(E, P, frames, positions, uniforms, **rule)


@pytest.mark.parametrize("V", [3, 100, 1025, 5000, 20000, 33000, 60000])
def test_sample_words_of_equal_and_masked_scores(V):
    E, P, frames, positions, g = make(4, 4, 2, V, 40, seed=V, holes=False)
    E[0], P[0] = 0.0, 0.0
    E[1], P[1] = (E[1] * 0.4).round(), P[1].round()
    E[2, :, torch.randperm(V, generator=g)[: V - max(1, V // 5)]] = -math.inf
    E[2, 1] = -math.inf
    E[2, 3] = torch.finfo(torch.float32).min
    E[3, 0, V // 2] = math.nan
    E[3, 1, V - 1] = math.inf
    uniforms = torch.rand(4, 40, generator=g).cuda()
    uniforms[:, 0], uniforms[:, 1], uniforms[:, 2] = -0.5, 1.5, math.nan
    for rule in RULES:
        check_sample(E, P, frames, positions, uniforms, **rule)


def test_sample_words_frequencies():
    """Shares of the words among evenly spaced numbers are their probabilities."""
    V, N = 50, 20000
    E, P, _, _, _ = make(1, 1, 1, V, 1)
    zero = torch.zeros(1, N, dtype=torch.int32).cuda()
    uniforms = ((torch.arange(N) + 0.5) / N)[None].cuda()
    words, log_probs = sample_words(E, P, zero, zero, uniforms)
    p = torch.softmax((E[0, 0] + P[0, 0]).double(), 0)
    share = torch.bincount(words[0].long(), minlength=V).double() / N
    assert (share - p).abs().max() <= 1.0 / N + 1e-9
    torch.testing.assert_close(log_probs[0].double(), p.log()[words[0].long()], rtol=0, atol=1e-5)


def teacher(E, P, frames, positions, K, g, temperature=1.0):
    Et = E.detach().float() + 0.7 * torch.randn(E.shape, generator=g).cuda()
    return top_words(Et, P.detach().float(), frames, positions, K, temperature)


def check_distill(E, P, frames, positions, words, logits, rest, temperature, g, K):
    E.requires_grad_(True)
    P.requires_grad_(True)
    weights = torch.randn(frames.shape, generator=g).cuda()
    criterion = NodeDistillationLoss(temperature=temperature)
    costs = criterion(E, P, frames, positions, words, logits, rest)
    dE, dP = torch.autograd.grad(costs, (E, P), weights)
    with torch.no_grad():
        assert torch.equal(costs, criterion(E, P, frames, positions, words, logits, rest))
    z, here = ref.scores(E, P, frames, positions)
    c, g64, cost_bound, grad_bound = ref.distill(z, here, words, logits, rest, temperature)
    got = costs.detach().cpu().double()
    finite = c.isfinite()
    assert torch.equal(got[~finite], c[~finite])
    assert ((got - c).abs()[finite] <= UNIT * cost_bound[finite]).all()
    w = weights.cpu().double()[..., None]
    de, dp = ref.spread(E, P, frames, positions, here, w * g64)
    # additions of a row's nodes: one more rounding of the sum so far for each
    me, mp = ref.spread(E, P, frames, positions, here, w.abs() * (grad_bound + frames.shape[1] * g64.abs()))
    half = torch.finfo(E.dtype).eps / 2 if E.dtype is torch.bfloat16 else 0.0
    for name, x, want, bound in (("dE", dE, de, me), ("dP", dP, dp, mp)):
        off = (x.cpu().double() - want).abs()
        allowed = UNIT * bound + half * (want.abs() + UNIT * bound) + 1e-37
        assert (off <= allowed).all(), (name, (off / allowed).max())
    again = torch.autograd.grad(criterion(E, P, frames, positions, words, logits, rest), (E, P), weights)
    assert torch.equal(again[0], dE) and torch.equal(again[1], dP)
    return costs, dE, dP


@pytest.mark.parametrize("V", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("kind", ["any", "path"])
def test_distillation(V, dtype, with_rest, kind):
    K = min(V, (1, 6, 33, 70)[V % 4])
    temperature = (1.0, 2.0, 0.5)[V % 3]
    E, P, frames, positions, g = make(2, 7, 4, V, 13, dtype, seed=V, kind=kind)
    words, logits, rest = teacher(E, P, frames, positions, K, g, temperature)
    check_distill(E, P, frames, positions, words, logits, rest if with_rest else None, temperature, g, K)


@pytest.mark.parametrize("V,B,T,U,N", [(40, 1, 1, 1, 1), (64, 3, 300, 2, 302), (96, 2, 400, 90, 520),
                                       (50, 2, 3, 200, 230), (1032, 1, 200, 1, 260), (260, 2, 6, 5, 1000)])
@pytest.mark.parametrize("kind", ["any", "path"])
@pytest.mark.parametrize("with_rest", [False, True])
def test_distillation_long_groups(V, B, T, U, N, kind, with_rest):
    """One position with many frames, many positions on few frames, frames without nodes."""
    E, P, frames, positions, g = make(B, T, U, V, N, seed=N, kind=kind, holes=N > 1)
    words, logits, rest = teacher(E, P, frames, positions, 5, g)
    check_distill(E, P, frames, positions, words, logits, rest if with_rest else None, 1.0, g, 5)


@pytest.mark.parametrize("scale,offset", [(300.0, 0.0), (1.0, 3e5), (1.0, -2e6), (50.0, 4e8), (1e33, 0.0)])
@pytest.mark.parametrize("V", [264, 1025, 3000])
@pytest.mark.parametrize("kind", ["any", "path"])
@pytest.mark.parametrize("with_rest", [False, True])
def test_distillation_of_wide_scores(scale, offset, V, kind, with_rest):
    """Scores of any size, rows that start masked and rows that rise from word to word."""
    E, P, frames, positions, g = make(2, 9, 3, V, 14, seed=V, kind=kind, holes=False)
    E = E * scale + offset
    E[0] = E[0].sort(-1).values
    E[1, :, :V // 2] = -math.inf
    words = torch.randint(0, V, (2, 14, 5), generator=g).int().cuda()
    words[1] = words[1] // 2 + V // 2
    logits = torch.randn(2, 14, 5, generator=g).cuda()
    rest = torch.randn(2, 14, generator=g).cuda()
    check_distill(E, P, frames, positions, words, logits, rest if with_rest else None, 1.5, g, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 1e-30, 1e20])
@pytest.mark.parametrize("V", [264, 1025])
@pytest.mark.parametrize("with_rest", [False, True])
def test_distillation_at_the_ends_of_the_range(dtype, temperature, V, with_rest):
    """Rows of the type's lowest number along a path, temperatures that leave one word or make all alike."""
    E, P, frames, positions, g = make(2, 9, 3, V, 14, dtype, seed=V, kind="path", holes=False)
    lowest = torch.finfo(dtype).min
    E[0, 1] = lowest
    E[0, 2, 5:] = lowest
    E[1, 3, :V // 2] = lowest
    words, logits, _ = top_words(E, P, frames, positions, 4)
    rest = torch.randn(2, 14, generator=g).cuda()
    check_distill(E, P, frames, positions, words, logits, rest if with_rest else None, temperature, g, 4)


def test_distillation_with_a_very_large_alphabet():
    E, P, frames, positions, g = make(1, 2, 1, (1 << 20) + 5, 3, holes=False)
    words, logits, rest = teacher(E, P, frames, positions, 7, g)
    check_distill(E, P, frames, positions, words, logits, rest, 1.0, g, 7)


@pytest.mark.parametrize("off", [(0,), (31, 32), (69,), (5, 40, 64, 65), tuple(range(70))])
def test_distillation_of_many_utterances_some_off_path(off):
    E, P, frames, positions, g = make(70, 6, 3, 40, 10, seed=len(off), kind="path")
    frames[list(off)] = frames[list(off)].flip(1)
    words, logits, rest = teacher(E, P, frames, positions, 4, g)
    check_distill(E, P, frames, positions, words, logits, rest, 1.0, g, 4)


@pytest.mark.parametrize("V", [30, 64, 1025])
@pytest.mark.parametrize("gap", [10, 100])
def test_distillation_paths_with_gaps(V, gap):
    """Paths of very different lengths, with runs of places that hold no node and frames without any."""
    E, P, frames, positions, g = make(4, 500, 6, V, 620, seed=V + gap, kind="path", holes=False)
    frames[0, 60:] = -1           # 60 of 500 frames have nodes
    frames[1] = -1                # none has
    frames[2, 200:200 + gap] = -1
    frames[3, :400] = -1          # the first frames have none
    frames[3, 500:500 + gap] = -1
    words, logits, rest = teacher(E, P, frames, positions, 5, g)
    check_distill(E, P, frames, positions, words, logits, rest, 1.0, g, 5)


@pytest.mark.parametrize("V", [30, 512, 1025, 5000])
@pytest.mark.parametrize("with_rest", [False, True])
def test_distillation_odd_records(V, with_rest):
    """Words listed twice, ignored ones, no record, teachers and students that mask words."""
    K = 12
    E, P, frames, positions, g = make(2, 8, 3, V, 14, seed=V, holes=False)
    words, logits, rest = teacher(E, P, frames, positions, K, g)
    words[0, 0, 3] = words[0, 0, 1]
    words[0, 0, 7] = words[0, 0, 1]
    words[0, 1, ::2] = -1
    words[0, 2] = -1
    rest[0, 2] = -math.inf
    logits[0, 3] = -math.inf
    rest[0, 3] = -math.inf
    logits[0, 4, 5:] = -math.inf
    rest[0, 5] = -math.inf
    rest[0, 6] += 60.0      # nearly all on words that are not listed
    logits[0, 7, 0] += 200.0
    # the student: on frame 6 the words that the teacher does not list are masked, on frame 7 all are
    frames[1] = torch.arange(14) % 6
    frames[1, 0], frames[1, 1], frames[1, 2] = 6, 7, 5
    E[1, 6] = -math.inf
    E[1, 6, words[1, 0].long()] = torch.randn(K, generator=g).cuda()
    E[1, 7] = -math.inf
    E[1, 5, words[1, 2, 0].long()] = -math.inf
    E[1, 4] = torch.finfo(torch.float32).min
    check_distill(E, P, frames, positions, words, logits, rest if with_rest else None, 1.0, g, K)


@pytest.mark.parametrize("with_rest", [False, True])
@pytest.mark.parametrize("K", [33, 64, 100, 256])
def test_distillation_long_records(K, with_rest):
    """Records of several words per lane, some longer than the vocabulary, with words more than once."""
    for V in (50, 300, 3001):
        E, P, frames, positions, g = make(2, 20, 4, V, 24, seed=K, kind="path")
        words = torch.randint(-1, V, (2, 24, K), generator=g).int().cuda()
        logits = (2.0 * torch.randn(2, 24, K, generator=g)).cuda()
        rest = torch.randn(2, 24, generator=g).cuda()
        check_distill(E, P, frames, positions, words, logits, rest if with_rest else None, 1.5, g, K)


def test_native_calls_without_optional_buffers():
    """No rest from the best words, no state from the forward call, one gradient alone."""
    from transducer_b200 import _transducer, nodes
    E, P, frames, positions, g = make(2, 9, 4, 100, 12, kind="path")
    words, logits, rest = top_words(E, P, frames, positions, 5)
    costs = NodeDistillationLoss()(E.requires_grad_(True), P.requires_grad_(True), frames, positions, words,
                                   logits + 0.3 * torch.randn(logits.shape, generator=g).cuda(), rest)
    weights = torch.rand(2, 12, generator=g).cuda()
    dE, dP = torch.autograd.grad(costs, (E, P), weights, retain_graph=True)
    saved = costs.grad_fn.saved_tensors[-1]
    with nodes.OnDevice(E.device):
        scores, sizes = nodes._describe(E, P, frames)
        at = frames.data_ptr(), positions.data_ptr()
        w2, l2 = torch.empty_like(words), torch.empty_like(logits)
        _transducer.top_words(scores, *at, w2.data_ptr(), l2.data_ptr(), 0, sizes, 5, 1.0)
        assert torch.equal(w2, words) and torch.equal(l2, logits)
        n = _transducer.distill_backward_workspace_bytes(*sizes)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        for which, want in ((0, dE), (1, dP)):
            out = torch.full_like(want, math.nan)
            to = (out.data_ptr(), 0) if which == 0 else (0, out.data_ptr())
            _transducer.distill_backward(scores, *at, words.data_ptr(), saved.data_ptr(), saved.numel(),
                                         weights.data_ptr(), *to, sizes, 5, 1.0, ws.data_ptr(), n)
            assert torch.equal(out, want)


@pytest.mark.parametrize("which", [0, 1, (0, 1)])
def test_second_derivatives_are_refused(which):
    E, P, frames, positions, g = make(2, 6, 4, 40, 9, holes=False)
    words, logits, rest = teacher(E, P, frames, positions, 4, g)
    E.requires_grad_(True), P.requires_grad_(True)
    leaves = [(E, P)[i] for i in (which if isinstance(which, tuple) else (which,))]
    cost = NodeDistillationLoss(reduction="sum")(E, P, frames, positions, words, logits, rest)
    plain = torch.autograd.grad(cost, leaves, retain_graph=True)
    grads = torch.autograd.grad(cost, leaves, create_graph=True)
    for a, b in zip(plain, grads):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (cost + sum(x.square().sum() for x in grads)).backward()


def test_the_same_tensor_on_both_sides():
    """Scores that are twice a row of one tensor: its gradient is both sides' together."""
    E, _, frames, positions, g = make(2, 6, 6, 40, 9, holes=False)
    words, logits, _ = teacher(E, E, frames, positions, 4, g)
    E.requires_grad_(True)
    other = E.detach().clone().requires_grad_(True)
    criterion = NodeDistillationLoss()
    both = torch.autograd.grad(criterion(E, E, frames, positions, words, logits).sum(), E)[0]
    a, b = torch.autograd.grad(criterion(E, other, frames, positions, words, logits).sum(), (E, other))
    torch.testing.assert_close(both, a + b, rtol=0, atol=0)


def test_distillation_where_every_word_is_listed():
    E, P, frames, positions, g = make(2, 5, 3, 20, 9)
    words, logits, rest = teacher(E, P, frames, positions, 20, g)
    assert (rest == -math.inf).all()
    check_distill(E, P, frames, positions, words, logits, rest, 1.0, g, 20)


def test_one_listed_word_is_minus_log_probability():
    E, P, frames, positions, g = make(2, 9, 4, 77, 12, holes=False)
    uniforms = torch.rand(2, 12, generator=g).cuda()
    words, log_probs = sample_words(E, P, frames, positions, uniforms)
    costs = NodeDistillationLoss()(E, P, frames, positions, words[..., None], torch.zeros(2, 12, 1).cuda())
    torch.testing.assert_close(costs, -log_probs, rtol=1e-5, atol=1e-5)


def test_gradients_against_differences():
    """Central differences of the costs in 64 bits, in random directions."""
    E, P, frames, positions, g = make(2, 6, 4, 37, 11, kind="path")
    words, logits, rest = teacher(E, P, frames, positions, 6, g)
    E.requires_grad_(True)
    P.requires_grad_(True)
    costs = NodeDistillationLoss()(E, P, frames, positions, words, logits, rest)
    dE, dP = torch.autograd.grad(costs.sum(), (E, P))
    b = torch.arange(2)[:, None].expand(frames.shape)
    here = (frames >= 0).cpu()

    def cost(e, p):
        z = torch.zeros(2, 11, 37, dtype=torch.float64)
        z[here] = e[b[here], frames.cpu()[here].long()] + p[b[here], positions.cpu()[here].long()]
        return ref.distill(z, here, words, logits, rest)[0].sum()

    e, p = E.detach().cpu().double(), P.detach().cpu().double()
    for _ in range(5):
        ve = torch.randn(e.shape, generator=g, dtype=torch.float64)
        vp = torch.randn(p.shape, generator=g, dtype=torch.float64)
        h = 1e-4
        slope = (cost(e + h * ve, p + h * vp) - cost(e - h * ve, p - h * vp)) / (2 * h)
        mine = (dE.cpu().double() * ve).sum() + (dP.cpu().double() * vp).sum()
        # (third derivatives times h^2, and the gradients' own rounding)
        assert abs(slope - mine) <= 1e-5 * max(1.0, abs(slope))


def test_layouts():
    """Time-major scores, slices, rows on odd addresses, expanded predictions: the same results."""
    E, P, frames, positions, g = make(3, 6, 4, 264, 10)
    uniforms = torch.rand(3, 10, generator=g).cuda()

    def all_of(E, P):
        E, P = E.detach().requires_grad_(True), P.detach().requires_grad_(True)
        words, logits, rest = top_words(E, P, frames, positions, 9)
        drawn = sample_words(E, P, frames, positions, uniforms, top_p=0.9)
        costs = NodeDistillationLoss()(E, P, frames, positions, words, logits, rest)
        return [words, logits, rest, *drawn, costs.detach(), *torch.autograd.grad(costs.sum(), (E, P))]

    want = all_of(E, P)
    time_major = E.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(3, 6, 301, device="cuda")
    wide[..., 5:269] = E
    words_first = E.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    flat = torch.zeros(P.numel() + 1, device="cuda")
    flat[1:] = P.flatten()
    for e, p in ((time_major, P), (wide[..., 5:269], P), (words_first, P), (E, flat[1:].view(P.shape))):
        for a, w in zip(all_of(e, p), want):
            torch.testing.assert_close(a, w, rtol=1e-5, atol=1e-6)
    one = P[:1].clone()
    P3 = one.expand(3, -1, -1)
    for a, w in zip(all_of(E, P3), all_of(E, P3.contiguous())):
        torch.testing.assert_close(a, w, rtol=1e-6, atol=1e-7)
    one.requires_grad_(True)
    words, logits, rest = top_words(E, P3, frames, positions, 9)
    costs = NodeDistillationLoss()(E, one.expand(3, -1, -1), frames, positions, words, logits - 1.0)
    assert torch.autograd.grad(costs.sum(), one)[0].shape == one.shape


def test_indices_beyond_the_tensors_are_no_nodes_when_not_validated():
    E, P, frames, positions, g = make(2, 4, 3, 50, 6, holes=False)
    words, logits, _ = top_words(E, P, frames, positions, 4)
    frames[0, 0], positions[0, 1], frames[1, 2], positions[1, 3] = 4, 3, -7, 2 ** 31 - 1
    words[1, 0, 0], words[1, 1] = 50, 2 ** 31 - 1
    with pytest.raises(ValueError, match="Frame index mismatch"):
        top_words(E, P, frames, positions, 4)
    w, l, r = top_words(E, P, frames, positions, 4, validate_nodes=False)
    z, here = ref.scores(E, P, frames, positions)
    assert here.sum() == 8 and torch.equal(w.cpu(), ref.top_words(z, here, 4)[0])
    drawn, log_probs = sample_words(E, P, frames, positions, torch.rand(2, 6).cuda(), validate_nodes=False)
    assert (drawn[~here.cuda()] == -1).all() and (log_probs[~here.cuda()] == 0).all()
    E.requires_grad_(True)
    costs = NodeDistillationLoss(validate_nodes=False)(E, P, frames, positions, words, logits)
    c, g64, _, _ = ref.distill(z, here, words, logits)
    torch.testing.assert_close(costs.detach().cpu().double(), c, rtol=1e-5, atol=1e-5)
    dE = torch.autograd.grad(costs.sum(), E)[0]
    torch.testing.assert_close(dE.cpu().double(), ref.spread(E, P, frames, positions, here, g64)[0],
                               rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("N", [1, 7, 40000])
def test_validated_indices(N):
    """Each index beyond its tensor is refused, wherever it is, and the next call is not affected."""
    E, P, frames, positions, g = make(2, 4, 3, 20, N, holes=False)
    words, logits, _ = top_words(E, P, frames, positions, 2)
    good = sample_words(E, P, frames, positions, torch.zeros(2, N).cuda())
    criterion = NodeDistillationLoss()
    for index, most, message in ((frames, 4, "Frame"), (positions, 3, "Position"), (words, 20, "Word")):
        flat = index.view(-1)
        for at in (0, flat.numel() // 2, flat.numel() - 1):
            was = flat[at].item()
            flat[at] = most
            if index is not words:
                with pytest.raises(ValueError, match=message + " index mismatch"):
                    top_words(E, P, frames, positions, 2)
                with pytest.raises(ValueError, match=message + " index mismatch"):
                    sample_words(E, P, frames, positions, torch.zeros(2, N).cuda())
            with pytest.raises(ValueError, match=message + " index mismatch"):
                criterion(E, P, frames, positions, words, logits)
            flat[at] = was
    again = sample_words(E, P, frames, positions, torch.zeros(2, N).cuda())
    assert all(torch.equal(a, b) for a, b in zip(good, again))


def test_masked_places_are_not_read():
    """NaN in rows without nodes and in nodes that are not weighted by the record stay there."""
    E, P, frames, positions, g = make(2, 5, 3, 40, 7, holes=False)
    frames[:, 3] = -1
    frames[frames == 4] = 1
    words, logits, rest = top_words(E, P, frames, positions, 4)
    E[:, 4] = math.nan
    logits[:, 3] = math.nan
    rest[:, 3] = math.nan
    costs, dE, dP = check_distill(E, P, frames, positions, words, logits, rest, 1.0, g, 4)
    assert dE.isfinite().all() and dP.isfinite().all() and (dE[:, 4] == 0).all()


@pytest.mark.parametrize("B,T,U,N", [(0, 3, 2, 4), (2, 3, 2, 0), (2, 0, 2, 4), (2, 3, 0, 4)])
def test_nothing_to_do(B, T, U, N):
    E = torch.zeros(B, T, 8, device="cuda", requires_grad=True)
    P = torch.zeros(B, U, 8, device="cuda", requires_grad=True)
    nodes = torch.full((B, N), -1, dtype=torch.int32, device="cuda")
    words, logits, rest = top_words(E, P, nodes, nodes, 3)
    assert words.shape == (B, N, 3) and (words == -1).all()
    drawn, _ = sample_words(E, P, nodes, nodes, torch.zeros(B, N, device="cuda"))
    assert (drawn == -1).all()
    costs = NodeDistillationLoss()(E, P, nodes, nodes, words, logits, rest)
    dE, dP = torch.autograd.grad(costs.sum(), (E, P))
    assert (costs == 0).all() and (dE == 0).all() and (dP == 0).all()
    assert NodeDistillationLoss(reduction="mean")(E, P, nodes, nodes, words, logits) == 0


def test_one_leaf_only():
    E, P, frames, positions, g = make(2, 5, 3, 40, 7)
    words, logits, _ = teacher(E, P, frames, positions, 4, g)
    E1, P1 = E.clone().requires_grad_(True), P.clone().requires_grad_(True)
    criterion = NodeDistillationLoss(reduction="sum")
    both = torch.autograd.grad(criterion(E1, P1, frames, positions, words, logits), (E1, P1))
    assert torch.equal(torch.autograd.grad(criterion(E1, P, frames, positions, words, logits), E1)[0], both[0])
    assert torch.equal(torch.autograd.grad(criterion(E, P1, frames, positions, words, logits), P1)[0], both[1])


def test_reductions():
    E, P, frames, positions, g = make(2, 5, 3, 40, 7)
    words, logits, _ = teacher(E, P, frames, positions, 4, g)
    costs = NodeDistillationLoss()(E, P, frames, positions, words, logits)
    total = NodeDistillationLoss(reduction="sum")(E, P, frames, positions, words, logits)
    mean = NodeDistillationLoss(reduction="mean")(E, P, frames, positions, words, logits)
    assert torch.equal(total, costs.sum())
    torch.testing.assert_close(mean, costs.sum() / (frames >= 0).sum())


def test_together_on_another_stream_and_in_a_graph():
    """A teacher's record on a path that the student drew, the student's step on it: eagerly on a
    stream of its own, and captured and replayed on new inputs."""
    E, P, frames, positions, g = make(4, 30, 6, 1000, 36, kind="path")
    Et, Pt = E + 0.5 * torch.randn(E.shape, generator=g).cuda(), P.clone()
    uniforms = torch.rand(4, 36, generator=g).cuda()
    criterion = NodeDistillationLoss(temperature=2.0, validate_nodes=False)

    def step(E, P):
        drawn, log_probs = sample_words(E, P, frames, positions, uniforms, top_k=50, validate_nodes=False)
        words, logits, rest = top_words(Et, Pt, frames, positions, 16, 2.0, validate_nodes=False)
        costs = criterion(E, P, frames, positions, words, logits, rest)
        return [drawn, log_probs, costs.detach(), *torch.autograd.grad(costs.sum(), (E, P))]

    E.requires_grad_(True)
    P.requires_grad_(True)
    want = step(E, P)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step(E, P)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    E2, P2 = E.detach().clone().requires_grad_(True), P.detach().clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(E2, P2)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        E2.mul_(0.5)
        E.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, step(E, P)))


def test_decoding_step_by_step():
    """Greedy decoding, a hypothesis per utterance: each step's words are the joiner's best ones."""
    E, P, _, _, _ = make(3, 12, 9, 130, 1)
    frames = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    labels = torch.zeros(3, dtype=torch.long, device="cuda")
    zero = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    numbers = torch.zeros(3, 1, device="cuda")
    for _ in range(20):
        rows = P[torch.arange(3, device="cuda"), labels][:, None]
        words, _ = sample_words(E, rows, frames, zero, numbers, temperature=0.0)
        there = frames[:, 0] < 12
        z = E[torch.arange(3, device="cuda"), frames[:, 0].clamp(max=11).long()] + rows[:, 0]
        assert torch.equal(words[there, 0].long(), z.argmax(-1)[there])
        blank = words[:, 0] % 3 == 0   # (a third of the words ends the frame here)
        frames = torch.where(blank[:, None] & (frames < 11), frames + 1, frames)
        labels = torch.where(blank, labels, (labels + 1).clamp(max=8))


def test_long_offsets():
    """Rows beyond 2^31 words from the start of the tensors."""
    V = 32000
    T = 2 ** 31 // V + 40
    E = torch.zeros(1, T, V, device="cuda", dtype=torch.bfloat16)
    E[0, -1] = torch.randn(V, generator=torch.Generator().manual_seed(3)).bfloat16()
    P = torch.zeros(1, 1, V, device="cuda", dtype=torch.bfloat16)
    frames = torch.tensor([[0, T - 1]], dtype=torch.int32, device="cuda")
    positions = torch.zeros_like(frames)
    words, logits, rest = top_words(E, P, frames, positions, 7)
    last = E[0, -1].float().cpu()
    assert torch.equal(words[0, 1].cpu(), torch.sort(last, descending=True, stable=True).indices[:7].int())
    E.requires_grad_(True)
    costs = NodeDistillationLoss()(E, P, frames, positions, words, logits - 1.0)
    dE = torch.autograd.grad(costs.sum(), E)[0]
    p = torch.softmax(last.double(), 0)
    q = torch.softmax(logits[0, 1].cpu().double(), 0)
    p[words[0, 1].cpu().long()] -= q
    torch.testing.assert_close(dE[0, -1].cpu().double(), p, rtol=2.0 ** -8 * 1.01, atol=1e-6)
    assert (dE[0, 1:-1] == 0).all()


def test_the_loss_beside_it_is_untouched():
    """The costs of the whole lattice before and after calls on its nodes."""
    E, P, frames, positions, g = make(2, 20, 5, 64, 9)
    labels = torch.randint(1, 64, (2, 4), generator=g).int().cuda()
    lens = torch.tensor([20, 15], dtype=torch.int32).cuda(), torch.tensor([4, 2], dtype=torch.int32).cuda()
    criterion = TransducerLoss()
    before = criterion(E, P, labels, *lens)
    top_words(E, P, frames, positions, 4)
    sample_words(E, P, frames, positions, torch.rand(2, 9, generator=g).cuda())
    assert torch.equal(before, criterion(E, P, labels, *lens))
