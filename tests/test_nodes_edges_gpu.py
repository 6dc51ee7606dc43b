"""Node operators (transducer_b200.nodes) at the edges of what their documentation allows."""
import math

import pytest
import torch

import node_reference as ref
from test_nodes_gpu import UNIT, check_distill, check_sample, make, teacher
from transducer_b200 import NodeDistillationLoss, TransducerLoss, sample_words, top_words

pytestmark = pytest.mark.gpu


# ---- draws among words of next to no weight ---------------------------------------------------

def test_draw_of_the_first_word_however_small():
    """A number of 0 takes the first word that has any weight in 64 bits, 2^-130 of the best one's here."""
    E = torch.tensor([[[-9.0, 0.0, -0.1]]]).cuda()
    zero = torch.zeros(1, 1, dtype=torch.int32).cuda()
    word, log_prob = sample_words(E, torch.zeros_like(E), zero, zero, torch.zeros(1, 1).cuda(), temperature=0.1)
    assert word.item() == 0
    z = torch.tensor([-9.0, 0.0, torch.tensor(-0.1).item()], dtype=torch.float64) / 0.1
    assert abs(log_prob.item() - torch.log_softmax(z, 0)[0].item()) <= 100 * 2 * UNIT


SMALL_RULES = [dict(), dict(top_k=2), dict(top_k=17), dict(top_k=400), dict(min_p=1e-30), dict(min_p=1e-40),
               dict(min_p=1e-200), dict(top_k=40, min_p=1e-60), dict(top_p=0.99), dict(top_k=30, top_p=0.9)]


@pytest.mark.parametrize("V", [3, 100, 520, 1025, 5000, 20000, 60000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_draws_with_the_smallest_numbers(V, dtype):
    """Temperatures at which most words have weights below 2^-126, and numbers down to 0."""
    N = 12
    E, P, frames, positions, g = make(2, 6, 4, V, N, dtype, seed=V + 2, holes=False)
    numbers = torch.tensor([0.0, 1e-45, 1e-42, 1e-38, 1e-35, 1e-30, 1e-20, 1e-8, 0.5, 1.0 - 2.0 ** -24, 0.0, 0.0])
    uniforms = numbers[torch.stack([torch.randperm(N, generator=g) for _ in range(2)])].cuda()
    for temperature in (0.3, 0.1, 0.04):
        for rule in SMALL_RULES:
            check_sample(E, P, frames, positions, uniforms, temperature=temperature, **rule)


# ---- alphabets beyond the whole numbers of 32-bit floats ----------------------------------------

def test_top_k_beyond_the_whole_numbers_of_32_bit_floats():
    """2^24 words of weight 1 and, after them, others that fall: the k first are the k best."""
    ones, falling = 2 ** 24, 40000
    E = torch.zeros(1, 1, ones + falling)
    E[0, 0, ones:] = -0.01 - 1e-5 * torch.arange(falling)
    upto = ones + torch.cumsum(E[0, 0, ones:].double().exp(), 0)
    P, zero = torch.zeros_like(E).cuda(), torch.zeros(1, 1, dtype=torch.int32).cuda()
    E = E.cuda()
    u = 1.0 - 2.0 ** -24
    for more in (12344, 12345, 12346, 12347, 20001, 20003, 30007, 39999):
        total = upto[more - 1].item()
        want = int((upto[:more] <= u * total).sum())
        assert (upto[:more] - u * total).abs().min() > 1e-3   # (64-bit sums are good to 1e-5 here)
        word, _ = sample_words(E, P, zero, zero, torch.full((1, 1), u).cuda(), top_k=ones + more)
        assert word.item() == ones + want, more


# ---- long lists over short rows ------------------------------------------------------------------

@pytest.mark.parametrize("V", [513, 514, 520, 600, 640, 768, 776, 1000, 1025, 1032])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [65, 190, 196, 197, 256])
@pytest.mark.parametrize("kind", ["spread", "equal", "masked", "broken"])
def test_long_lists_over_short_rows(V, dtype, k, kind):
    E, P, frames, positions, g = make(2, 5, 3, V, 9, dtype, seed=V + k, holes=False)
    if kind == "equal":
        E, P = E.round(), P.round()
        E[0], P[0] = 0.0, 0.0
    elif kind == "masked":
        E[0, :, torch.randperm(V, generator=g)[k - 10:]] = -math.inf
        E[1, :, torch.randperm(V, generator=g)[:V - k]] = torch.finfo(dtype).min
    elif kind == "broken":
        E[0, 1, V // 3], E[0, 2, 5] = math.nan, math.inf
        E[1, 3, :k + 3] = math.nan
    words, logits, rest = top_words(E, P, frames, positions, k)
    z, here = ref.scores(E, P, frames, positions)
    w, l, r = ref.top_words(z, here, k)
    if kind == "broken":   # (NaN stands first: among NaN, and beside them, the order is the reference's)
        whole = z.isfinite().all(-1)
        assert whole.any() and not whole.all()
        assert torch.equal(words.cpu()[whole], w[whole])
        torch.testing.assert_close(rest.cpu().double()[whole], r[whole], rtol=64 * UNIT, atol=128 * UNIT)
        assert torch.equal(words.cpu(), w)
        torch.testing.assert_close(logits.cpu().double(), l, rtol=0, atol=0, equal_nan=True)
        return
    assert torch.equal(words.cpu(), w)
    assert torch.equal(logits.cpu().double(), l)
    torch.testing.assert_close(rest.cpu().double(), r, rtol=64 * UNIT, atol=128 * UNIT)


def microseconds(call, runs=15):
    times = []
    for _ in range(runs):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(1e3 * a.elapsed_time(b))
    return sorted(times[3:])[len(times[3:]) // 2]


def test_long_lists_over_short_rows_take_no_longer_than_over_longer_ones():
    """196 words of rows of 520 were found by going through the row from memory for every bit of a score, in 2.3 times
    the time of rows of twice the words (now 1.1)."""
    def time(V):
        E, P, frames, positions, _ = make(8, 60, 30, V, 1000, torch.bfloat16, seed=V, holes=False)
        return microseconds(lambda: top_words(E, P, frames, positions, 196, validate_nodes=False))
    assert time(520) <= 1.6 * time(1040)


# ---- shares that end at a gap ---------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [520, 1025, 10000, 20000, 60000])
@pytest.mark.parametrize("off", [-1e-7, -1e-9, -1e-12, 1e-12, 1e-9, 1e-7])   # (0: sums in 64 bits round)
def test_shares_next_to_the_sum_of_the_words_above_a_gap(V, dtype, off):
    """Twenty words have nearly all of the weight: the share is theirs, or a little less or more than 32 bits can tell."""
    E, top_p, frames, zero, uniforms = gap(V, dtype, 6, 1.0 + off)
    check_sample(E, torch.zeros_like(E), frames, zero, uniforms, top_p=top_p)


def gap(V, dtype, N, factor):
    g = torch.Generator().manual_seed(V)
    E = -9.0 - torch.rand(1, N, V, generator=g)
    for n in range(N):
        E[0, n, torch.randperm(V, generator=g)[:20]] = -torch.rand(20, generator=g)
    E[0, :] = E[0, :1]
    E = E.to(dtype)
    w = (E[0, 0].double() - E[0, 0].double().max()).exp().sort(descending=True).values
    frames = torch.arange(N)[None].int().cuda()
    top_p = (w[:20].sum() / w.sum()).item() * factor
    return E.cuda(), top_p, frames, torch.zeros_like(frames), torch.rand(1, N, generator=g).cuda()


def test_a_share_next_to_a_gap_is_found_as_fast_as_another():
    """64 rounds and 48 passes in 64 bits were made: 27 times as long as for another share (now 4)."""
    def time(factor):
        E, top_p, frames, zero, uniforms = gap(10000, torch.float32, 64, factor)
        P = torch.zeros_like(E)
        return microseconds(lambda: sample_words(E, P, frames, zero, uniforms, top_p=top_p, validate_nodes=False))
    assert max(time(1.0 - 1e-9), time(1.0 + 1e-9)) <= 10.0 * time(0.99)


# ---- bf16 gradients along a path whose scores are far from 0 -------------------------------------

@pytest.mark.parametrize("offset", [0.0, 120.0, 496.0, -496.0, 30000.0])
@pytest.mark.parametrize("temperature", [0.75, 1.0, 8.0])
@pytest.mark.parametrize("own_record", [True, False])
def test_bf16_paths_with_scores_far_from_0(offset, temperature, own_record):
    """Where the record is the student's own distribution the gradients are small differences, however far the scores
    are from 0: one node for each frame and position, so that nothing averages."""
    B, N, V, K = 4, 40, 16, 16 if own_record else 5
    g = torch.Generator().manual_seed(int(abs(offset)) + own_record)
    E = (offset + 2.0 * torch.randint(-2, 3, (B, N, V), generator=g)).bfloat16().cuda()
    P = torch.randn(B, N, V, generator=g).bfloat16().cuda()
    nodes = torch.arange(N).expand(B, N).contiguous().int().cuda()
    if own_record:
        words, logits, _ = top_words(E, P, nodes, nodes, K, temperature)
    else:
        words, logits, _ = teacher(E, P, nodes, nodes, K, g, temperature)
    check_distill(E, P, nodes, nodes, words, logits, None, temperature, g, K)


# ---- records that want gradients ---------------------------------------------------------

@pytest.mark.parametrize("student", [False, True])
@pytest.mark.parametrize("which", ["logits", "rest"])
def test_records_that_want_gradients_are_refused(student, which):
    E, P, frames, positions, g = make(2, 5, 3, 20, 7, holes=False)
    words, logits, rest = teacher(E, P, frames, positions, 4, g)
    E.requires_grad_(student)
    (logits if which == "logits" else rest).requires_grad_(True)
    criterion = NodeDistillationLoss()
    with pytest.raises(ValueError, match="not differentiable w.r.t. the teacher's record"):
        criterion(E, P, frames, positions, words, logits, rest)
    with torch.no_grad():
        costs = criterion(E, P, frames, positions, words, logits, rest)
    assert torch.equal(costs, criterion(E, P, frames, positions, words, logits.detach(), rest.detach()).detach())


# ---- what is not differentiable --------------------------------------------------------------------

def test_tangents_are_refused():
    from torch.autograd import forward_ad
    E, P, frames, positions, g = make(2, 5, 3, 20, 7, holes=False)
    words, logits, rest = teacher(E, P, frames, positions, 4, g)
    uniforms = torch.rand(2, 7, generator=g).cuda()
    with forward_ad.dual_level():
        top_words(E, P, frames, positions, 4)    # (no tangent)
        for e, p in ((forward_ad.make_dual(E, torch.ones_like(E)), P), (E, forward_ad.make_dual(P, torch.ones_like(P)))):
            with pytest.raises(RuntimeError, match="no tangents"):
                top_words(e, p, frames, positions, 4)
            with pytest.raises(RuntimeError, match="no tangents"):
                sample_words(e, p, frames, positions, uniforms)
            with pytest.raises(RuntimeError):
                NodeDistillationLoss()(e, p, frames, positions, words, logits, rest)


def test_best_words_and_draws_are_detached():
    E, P, frames, positions, g = make(2, 5, 3, 20, 7, holes=False)
    E.requires_grad_(True)
    assert not any(x.requires_grad for x in top_words(E, P, frames, positions, 4))
    assert not any(x.requires_grad for x in sample_words(E, P, frames, positions, torch.rand(2, 7, generator=g).cuda()))


# ---- batches of small lattices -------------------------------------------------------------------

def lattices(B, T, U, V, dtype, seed):
    E, P, _, _, g = make(B, T, U, V, 1, dtype, seed=seed)
    frames = torch.arange(T)[:, None].expand(T, U).reshape(1, -1).expand(B, T * U).clone()
    positions = torch.arange(U)[None, :].expand(T, U).reshape(1, -1).expand(B, T * U).clone()
    frames[1, T * U // 2:] = -1
    return E, P, frames.int().cuda(), positions.int().cuda(), g


@pytest.mark.parametrize("B,T,U,V", [(32, 20, 5, 100), (33, 12, 6, 520), (1500, 2, 2, 24), (3, 40, 9, 1032)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distillation_of_many_lattices(B, T, U, V, dtype):
    E, P, frames, positions, g = lattices(B, T, U, V, dtype, seed=B)
    words, logits, rest = teacher(E, P, frames, positions, 4, g)
    check_distill(E, P, frames, positions, words, logits, rest, 1.0, g, 4)


def test_small_lattices_share_the_chip():
    """The gradients of thirty-two small lattices took thirteen times as long as those of one (now 1.2)."""
    from transducer_b200 import _transducer, nodes

    def time(B):
        E, P, frames, positions, g = lattices(32, 20, 5, 100, torch.float32, seed=3)
        E, P, frames, positions = (x[:B].contiguous() for x in (E, P, frames, positions))
        words, logits, rest = teacher(E, P, frames, positions, 4, g)
        costs = NodeDistillationLoss()(E.requires_grad_(True), P, frames, positions, words, logits, rest)
        saved = costs.grad_fn.saved_tensors[-1]
        weights, dE, dP = torch.ones_like(costs), torch.empty_like(E), torch.empty_like(P)
        with nodes.OnDevice(E.device):
            scores, sizes = nodes._describe(E, P, frames)
            n = _transducer.distill_backward_workspace_bytes(*sizes)
            ws = torch.empty(n, dtype=torch.uint8, device="cuda")

            def backward():
                for _ in range(5):
                    _transducer.distill_backward(
                        scores, frames.data_ptr(), positions.data_ptr(), words.data_ptr(), saved.data_ptr(),
                        saved.numel(), weights.data_ptr(), dE.data_ptr(), dP.data_ptr(), sizes, 4, 1.0, ws.data_ptr(), n)
            return microseconds(backward)
    assert time(32) <= 4.0 * time(1)


# ---- two-byte rows along paths of many segments ----------------------------------------------------

@pytest.mark.parametrize("V", [1032, 2051, 2568])
@pytest.mark.parametrize("gap", [10, 100])
@pytest.mark.parametrize("with_rest", [False, True])
def test_bf16_paths_of_many_segments(V, gap, with_rest):
    """As test_distillation_paths_with_gaps, in bf16, with rows of several tiles and turns of the ring, and nodes enough
    for a warp each."""
    E, P, frames, positions, g = make(4, 500, 6, V, 620, torch.bfloat16, seed=V + gap, kind="path", holes=False)
    frames[0, 60:] = -1
    frames[2, 200:200 + gap] = -1
    frames[3, :400] = -1
    words, logits, rest = teacher(E, P, frames, positions, 5, g)
    check_distill(E, P, frames, positions, words, logits, rest if with_rest else None, 1.0, g, 5)


@pytest.mark.parametrize("V,B,T,U,N", [(64, 3, 300, 2, 302), (96, 2, 400, 90, 520), (56, 2, 3, 200, 230),
                                       (1032, 1, 200, 1, 260), (520, 2, 90, 60, 150)])
@pytest.mark.parametrize("kind", ["any", "path"])
@pytest.mark.parametrize("K", [5, 40])
def test_bf16_long_groups(V, B, T, U, N, kind, K):
    """One position with many frames, many positions on few frames, in bf16."""
    E, P, frames, positions, g = make(B, T, U, V, N, torch.bfloat16, seed=N, kind=kind)
    words, logits, rest = teacher(E, P, frames, positions, K, g)
    check_distill(E, P, frames, positions, words, logits, rest, 1.0, g, K)


# ---- the nodes of an alignment -------------------------------------------------------------------

def test_nodes_of_an_alignment():
    """On one frame there is one alignment: its nodes' costs add up to the lattice's."""
    B, U, V = 3, 5, 40
    g = torch.Generator().manual_seed(8)
    E, P = torch.randn(B, 1, V, generator=g).cuda(), torch.randn(B, U + 1, V, generator=g).cuda()
    labels = torch.randint(1, V, (B, U), generator=g).int().cuda()
    lengths = torch.tensor([5, 0, 3]).cuda()
    moves = (torch.arange(U + 1, device="cuda") < lengths[:, None]).long()
    n_moves = lengths + 1
    n = torch.arange(moves.shape[1], device=moves.device)
    positions = moves.cumsum(1) - moves
    frames = n - positions
    gone = n >= n_moves[:, None]
    frames, positions = (x.masked_fill(gone, -1).int() for x in (frames, positions))
    words = torch.where(moves.bool(), torch.nn.functional.pad(labels, (0, 1)), 0).int()[..., None].contiguous()
    E.requires_grad_(True), P.requires_grad_(True)
    costs = NodeDistillationLoss()(E, P, frames, positions, words, torch.zeros(B, U + 1, 1).cuda())
    grads = torch.autograd.grad(costs.sum(), (E, P))
    whole = TransducerLoss()(E, P, labels, torch.ones(B, dtype=torch.int32).cuda(), lengths.int())
    torch.testing.assert_close(costs.sum(1), whole, rtol=1e-5, atol=1e-4)
    for a, b in zip(grads, torch.autograd.grad(whole.sum(), (E, P))):
        torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-4)
