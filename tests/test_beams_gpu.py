"""extend_beams, reorder_states and embed_words against their definitions in 64 bits."""
import math

import pytest
import torch

import beam_reference as ref
from transducer_b200 import TransducerLoss, embed_words, extend_beams, reorder_states

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24          # of a 32-bit rounding
TYPES = [torch.float32, torch.bfloat16]
INF = math.inf


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---- the best extensions ----------------------------------------------------------------------

def hypotheses(B, T, U, V, N, dtype=torch.float32, seed=0, done=0.15, gone=0.1, std=2.0):
    g = torch.Generator().manual_seed(seed)
    E = (std * torch.randn(B, T, V, generator=g)).to(dtype)
    P = torch.randn(B, U, V, generator=g).to(dtype)
    frames = torch.randint(0, T, (B, N), generator=g).int()
    positions = torch.randint(0, U, (B, N), generator=g).int()
    scores = -20.0 + 3.0 * torch.randn(B, N, generator=g)
    kind = torch.rand(B, N, generator=g)
    frames[kind < done / 2] = -1
    positions[(kind >= done / 2) & (kind < done)] = -1
    scores[kind > 1 - gone] = -INF
    return [x.cuda() for x in (E, P, frames, positions, scores)]


def check_extend(args, width, **options):
    got = extend_beams(*args, width, **options)
    want = ref.extend(*args, width)
    scores, parents, words = (x.cpu() for x in got)
    assert torch.equal(parents, want[1])
    assert torch.equal(words, want[2])
    # log-sum-exp in 32 bits is good to 6e-6 (the kernels' own bound); the result is rounded once
    d = want[0]
    assert torch.equal(scores.isnan(), d.isnan())
    assert torch.equal(scores == -INF, d == -INF)
    fine = d.isfinite()
    assert ((scores.double() - d).abs()[fine] <= 6e-6 + 1.01 * UNIT * d.abs()[fine]).all()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,N,width", [
    (1, 1, 1), (1, 3, 8), (2, 1, 5), (8, 4, 4), (31, 5, 8), (32, 5, 40), (33, 1, 33), (100, 70, 16), (264, 8, 64),
    (1000, 1, 256), (1023, 3, 8), (1024, 9, 100), (1025, 8, 8), (2049, 33, 32), (4096, 16, 256), (5000, 40, 1),
    (32000, 6, 8), (70001, 2, 12)])
def test_extensions(V, N, width, dtype):
    for seed in range(3):
        check_extend(hypotheses(3, 7, 5, V, N, dtype, seed=seed), width)


def test_many_hypotheses():
    check_extend(hypotheses(2, 4, 4, 24, 3000, seed=1), 200)
    check_extend(hypotheses(1, 3, 3, 1100, 400, torch.bfloat16, seed=2), 64)
    check_extend(hypotheses(300, 3, 3, 40, 2, seed=3), 4)


def test_one_hypothesis_far_ahead():
    """All extensions are of one row, and of a few words of it."""
    for V in (50, 1025, 9000):
        args = hypotheses(2, 4, 6, V, 12, seed=4, done=0.0, gone=0.0)
        args[4][:, 7] += 100.0
        check_extend(args, 48)
        args[0][:, :, V // 2] += 60.0
        check_extend(args, 48)


@pytest.mark.parametrize("V", [5, 1030, 40000])
@pytest.mark.parametrize("dtype", TYPES)
def test_equal_scores(V, dtype):
    """All words of all hypotheses are equally good: the order is that of the indices, also behind a finished one."""
    N = 6
    E, P = torch.zeros(2, 1, V, dtype=dtype), torch.zeros(2, 1, V, dtype=dtype)
    frames = positions = torch.zeros(2, N, dtype=torch.int32)
    scores = torch.full((2, N), -3.0)
    scores[1, 2] = -2.5
    args = [x.cuda() for x in (E, P, frames, positions, scores)]
    for width in (1, 7, 256):
        check_extend(args, width)
    args[2] = args[2].clone()
    args[2][:, 1] = -1
    args[4][:, 1] = -3.0 - torch.tensor(float(V)).log().item()   # (about as good as its neighbours' words)
    check_extend(args, 200)


def test_two_values():
    """More equal scores than any list holds, after a few better ones in the middle."""
    E = torch.zeros(1, 2, 30000)
    E[0, 0, 15000:15003] = 1.0
    E[0, 1, 20000] = 1.0
    P = torch.zeros(1, 1, 30000)
    frames = torch.tensor([[0, 1, 0, 1]], dtype=torch.int32)
    positions = torch.zeros(1, 4, dtype=torch.int32)
    scores = torch.tensor([[-1.0, -1.0, -1.0, -1.5]])
    for width in (2, 8, 100):
        check_extend([x.cuda() for x in (E, P, frames, positions, scores)], width)


@pytest.mark.parametrize("width", [1, 40, 64, 256])
def test_scores_that_lists_are_not_made_for(width):
    """Few values, values next to each other, values that rise, and good hypotheses a multiple of 8 apart."""
    V, N = 3000, 40
    E, P, frames, positions, scores = hypotheses(2, 4, N, V, N, seed=20, done=0.05, gone=0.0)
    positions[positions >= 0] = torch.arange(N, device="cuda").repeat(2, 1)[positions >= 0].int()
    few = torch.randint(0, 3, E.shape, generator=torch.Generator().manual_seed(1)).float().cuda()
    rising = torch.arange(V, device="cuda").expand_as(E).contiguous()
    flat = torch.full_like(scores, -5.0)
    for e, p, s in ((few, 0 * P, flat), (1e-7 * E, 1e-7 * P, flat), (few, 1e-7 * P, flat), (1e-6 * rising, 0 * P, flat),
                    (-1e-6 * rising, 0 * P, flat), (1e-3 * rising, 0 * P, flat), (0 * E, P, flat), (E, 0 * P, flat)):
        check_extend([e, p, frames, positions, s], width)
    check_extend([few, 0 * P, frames, positions, scores], width)
    ahead = scores.clone()
    ahead[:, ::8] += 30.0
    check_extend([E, P, frames, positions, ahead], width)
    ahead[:, 1:] -= 60.0
    check_extend([E, P, frames, positions, ahead], width)
    lowest = torch.full_like(P, torch.finfo(torch.float32).min)
    lowest[:, :, 5] = 0.0
    check_extend([E, lowest, frames, positions, scores], width)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_hypotheses(dtype):
    """The same node and score more than once: the lower parent first."""
    E, P, frames, positions, scores = hypotheses(2, 3, 3, 1500, 8, dtype, seed=5, done=0.0, gone=0.0)
    frames[:, 4:], positions[:, 4:], scores[:, 4:] = frames[:, :4], positions[:, :4], scores[:, :4]
    check_extend([E, P, frames, positions, scores], 30)


@pytest.mark.parametrize("gap", [1e-7, 1e-8, 1e-9, 1e-12])
@pytest.mark.parametrize("V", [40, 1025, 6000])
def test_closer_than_32_bits(gap, V):
    """Hypotheses that differ by one word so unlikely that only 64 bits tell their log-sum-exps apart."""
    N = 8
    g = torch.Generator().manual_seed(V)
    row = torch.randn(V, generator=g).double()
    lse = row.logsumexp(0)
    P = row.float().repeat(1, N, 1)
    order = torch.randperm(N, generator=g)
    P[0, torch.arange(N), V - 1] = (lse + ((1.0 + order) * gap).log()).float()
    zero = torch.zeros(1, N, dtype=torch.int32)
    args = [torch.zeros(1, 1, V), P, zero, torch.arange(N).int()[None], torch.full((1, N), -1.5)]
    want = ref.extend(*args, 5)
    assert want[1][0].tolist() == [order.tolist().index(i) for i in range(5)]   # (the smallest sum first)
    for width in (1, 5, 30):
        check_extend([x.cuda() for x in args], width)


def test_masks():
    V, N = 1200, 5
    for dtype in TYPES:
        lowest = torch.finfo(dtype).min
        for value in (-INF, lowest):
            E, P, frames, positions, scores = hypotheses(3, 4, N, V, N, dtype, seed=6, done=0.0, gone=0.0)
            positions[:] = torch.arange(N, device="cuda")
            P[0, 0] = value                      # nothing is left of a row
            P[0, 1, 3:] = value                  # three words
            P[1, :, 700:] = value                # tiles without a word
            P[1, 2, :1100] = value
            E[2] = value                         # nothing at all
            for width in (2, 8, 200):
                check_extend([E, P, frames, positions, scores], width)


def test_not_there_and_no_numbers():
    E, P, frames, positions, scores = hypotheses(6, 3, 4, 1100, 4, seed=7, done=0.0, gone=0.0)
    frames[:] = 0
    positions[:] = torch.arange(4, device="cuda")
    P[0, 1, 17] = math.nan          # a row that counts
    P[1, 2, 1099] = INF
    P[2, 3] = math.nan              # a row that does not
    scores[2, 3] = -INF
    scores[3, 0] = math.nan
    scores[4, 0] = INF
    frames[4, 0] = -1
    scores[5] = -INF                # nobody is there
    got = check_extend([E, P, frames, positions, scores], 6)
    assert got[0][[0, 1, 3, 4]].isnan().all() and got[0][2].isfinite().all() and (got[1][5] == -1).all()


def test_finished_hypotheses_alone():
    scores = torch.tensor([[-3.0, -1.0, -INF, -1.0, -2.0]]).cuda()
    none = torch.full((1, 5), -1, dtype=torch.int32).cuda()
    E = torch.full((1, 2, 9), math.nan).cuda()
    best, parents, words = check_extend([E, E, none, none, scores], 5)
    assert parents.tolist() == [[1, 3, 4, 0, -1]] and (words == -1).all()


def test_no_frames_and_no_hypotheses():
    args = hypotheses(2, 3, 3, 10, 0)
    best, parents, words = extend_beams(*args, 4)
    assert (best == -INF).all() and (parents == -1).all() and (words == -1).all()
    args = hypotheses(0, 3, 3, 10, 4)
    assert extend_beams(*args, 4)[0].shape == (0, 4)
    E, P, frames, positions, scores = hypotheses(2, 3, 3, 10, 4, done=0.0, gone=0.0)
    best, parents, words = extend_beams(E[:, :0], P, frames, positions, scores, 2, validate_nodes=False)
    assert (words == -1).all() and (parents >= 0).all()   # (no frame: they are finished)


def test_large_magnitudes():
    E, P, frames, positions, scores = hypotheses(2, 3, 3, 1500, 6, seed=8, done=0.2, gone=0.0)
    check_extend([E + 30000.0, P - 29990.0, frames, positions, scores * 1000.0], 20)
    check_extend([E * 1e30, P, frames, positions, scores * 1e30], 20)
    check_extend([E * 1e37, P * 1e37, frames, positions, scores * 1e37], 20)


def test_strides():
    E, P, frames, positions, scores = hypotheses(3, 4, 5, 1032, 6, seed=9)
    want = extend_beams(E, P, frames, positions, scores, 9)
    wide = torch.zeros(3, 9, 2064, device="cuda")
    e = wide[:, 1:9:2, 8:1040].copy_(E)              # aligned, not contiguous
    p = torch.zeros(5, 3, 1033, device="cuda")[:, :, 1:].copy_(P.transpose(0, 1)).transpose(0, 1)   # odd
    columns = torch.zeros(3, 1032, 4, device="cuda").transpose(1, 2).copy_(E)   # words apart
    for x in (e, columns):
        for y in (P, p):
            for a, b in zip(extend_beams(x, y, frames, positions, scores, 9)[1:], want[1:]):
                assert torch.equal(a, b)
            assert torch.allclose(extend_beams(x, y, frames, positions, scores, 9)[0], want[0], rtol=0, atol=2e-5)
    # a table of predictions for all utterances, by the last word
    table = P[:1].expand(3, 5, 1032)
    check_extend([E, table, frames, positions, scores], 9)


def test_far_offsets():
    """Rows whose first word is beyond 2^31 words, and beyond 2^32 bytes."""
    V, U = 32768, 70000
    P = torch.empty(1, U, V, dtype=torch.bfloat16, device="cuda")
    rows = [0, 1, 65535, 65536, 69999]
    g = torch.Generator().manual_seed(10)
    P[0, rows] = torch.randn(5, V, generator=g).bfloat16().cuda()
    E = torch.randn(1, 2, V, generator=g).bfloat16().cuda()
    frames = torch.tensor([[0, 1, 0, 1, 0]], dtype=torch.int32).cuda()
    scores = torch.tensor([[-1.0, -1.2, -0.9, -1.1, -1.05]]).cuda()
    got = extend_beams(E, P, frames, torch.tensor([rows], dtype=torch.int32).cuda(), scores, 12)
    small = P[:, rows].contiguous()
    check_extend([E, small, frames, torch.arange(5, dtype=torch.int32).cuda()[None], scores], 12)
    want = extend_beams(E, small, frames, torch.arange(5, dtype=torch.int32).cuda()[None], scores, 12)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_indices_beyond():
    E, P, frames, positions, scores = hypotheses(2, 3, 4, 20, 3, done=0.0, gone=0.0)
    frames[1, 2] = 3
    with pytest.raises(ValueError, match="Frame index mismatch"):
        extend_beams(E, P, frames, positions, scores, 2)
    check_extend([E, P, frames, positions, scores], 8, validate_nodes=False)   # (taken for none)
    frames[1, 2], positions[0, 0] = 0, 4
    with pytest.raises(ValueError, match="Position index mismatch"):
        extend_beams(E, P, frames, positions, scores, 2)


def test_nodes_of_hypotheses_that_are_not_there():
    """They are not looked at, nor checked; and a refused call leaves nothing behind for the next one."""
    E, P, frames, positions, scores = hypotheses(2, 3, 4, 20, 3, done=0.0, gone=0.0)
    for _ in range(3):
        frames[0, 1], positions[0, 1], scores[0, 1] = 2 ** 30, 2 ** 31 - 1, -INF
        check_extend([E, P, frames, positions, scores], 8)
        scores[0, 1] = -1.0
        with pytest.raises(ValueError, match="Frame index mismatch"):
            extend_beams(E, P, frames, positions, scores, 2)


def test_checked_calls_of_many_threads():
    """Each sees its own indices."""
    import threading
    E, P, frames, positions, scores = hypotheses(2, 3, 4, 200, 3, done=0.0, gone=0.0)
    bad = frames.clone()
    bad[1, 1] = 3
    wrong = []

    def call(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for k in range(30):
                refused = False
                try:
                    extend_beams(E, P, bad if (i + k) % 3 == 0 else frames, positions, scores, 2)
                except ValueError:
                    refused = True
                if refused != ((i + k) % 3 == 0):
                    wrong.append((i, k))
    torch.cuda.synchronize()
    threads = [threading.Thread(target=call, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_results_are_detached_and_the_same_from_run_to_run():
    args = hypotheses(4, 3, 4, 5000, 12, seed=11)
    args[0].requires_grad_(True)
    first = extend_beams(*args, 40)
    assert not any(x.requires_grad for x in first)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(extend_beams(*args, 40), first))


def test_other_streams_and_graphs():
    """A captured call sees what its inputs hold when it is replayed; two graphs may run side by side."""
    sets = [hypotheses(4, 3, 6, 3000, 6, seed=s) for s in range(4)]
    want = [extend_beams(*a, 10) for a in sets]
    held = [[x.clone() for x in sets[0]] for _ in range(2)]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a, stream in zip(held, side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(extend_beams(*a, 10, validate_nodes=False))
        graphs.append(graph)
    for turn in range(3):
        for i in range(2):
            for x, y in zip(held[i], sets[turn + i]):
                x.copy_(y)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, side):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(x, y) for x, y in zip(outs[i], want[turn + i]))


# ---- states that follow -----------------------------------------------------------------------

def plain_reorder(states, parents, out=None):
    made = []
    for i, s in enumerate(states):
        B, W = parents.shape
        o = torch.zeros((B, W) + tuple(s.shape[2:]), dtype=s.dtype) if out is None else out[i].cpu().clone()
        s = s.cpu().clone()
        for b in range(B):
            for w in range(W):
                n = parents[b, w].item()
                if 0 <= n < s.shape[1]:
                    o[b, w] = s[b, n]
        made.append(o)
    return made


def some_states(B, N, g):
    shapes = [(), (1,), (3,), (7,), (16,), (640,), (641,), (5, 33), (2, 4, 40), (2049,), (0,)]
    states = []
    for i, shape in enumerate(shapes):
        dtype = [torch.float32, torch.bfloat16, torch.int32, torch.uint8, torch.int64, torch.bool][i % 6]
        x = torch.randint(0, 2 if dtype is torch.bool else 200, (B, N) + shape, generator=g)
        states.append(x.to(dtype).cuda())
    return states


def some_parents(B, N, W, g):
    parents = torch.randint(0, N, (B, W), generator=g).int()
    parents[torch.rand(B, W, generator=g) < 0.2] = -1
    return parents.cuda()


@pytest.mark.parametrize("B,N,W", [(1, 1, 1), (2, 3, 3), (3, 8, 5), (4, 5, 12), (1, 64, 64), (33, 2, 3)])
def test_states(B, N, W):
    g = torch.Generator().manual_seed(B * N)
    states, parents = some_states(B, N, g), some_parents(B, N, W, g)
    got = reorder_states(states, parents)
    for a, b in zip(got, plain_reorder(states, parents)):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b)
    one = reorder_states(states[5], parents)
    assert torch.equal(one, got[5])
    out = [torch.ones_like(x) for x in got]
    before = [x.cpu() for x in out]
    assert all(a is b for a, b in zip(reorder_states(states, parents, out=out), out))
    for a, b in zip(out, plain_reorder(states, parents, before)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("B,N,W", [(1, 1, 1), (2, 3, 3), (3, 8, 5), (4, 5, 12), (2, 64, 64), (2, 3000, 3000), (1, 4096, 4096)])
def test_states_in_place(B, N, W):
    """The state itself, its first hypotheses, or more room than there were; identical rows are left alone."""
    g = torch.Generator().manual_seed(N + W)
    parents = some_parents(B, N, W, g)
    rooms = [torch.zeros((B, max(N, W)) + s.shape[2:], dtype=s.dtype, device="cuda") for s in some_states(B, N, g)]
    for room, s in zip(rooms, some_states(B, N, g)):
        room[:, :N] = s
    states, out = [r[:, :N] for r in rooms], [r[:, :W] for r in rooms]
    want = plain_reorder(states, parents, out)
    behind = [r[:, W:].cpu().clone() for r in rooms]
    versions = [o._version for o in out]
    reorder_states(states, parents, out=out)
    for a, b, r, rest, v in zip(out, want, rooms, behind, versions):
        assert torch.equal(a.cpu(), b) and torch.equal(r[:, W:].cpu(), rest) and a._version > v


def test_many_states_and_strides():
    g = torch.Generator().manual_seed(3)
    B, N, W = 3, 6, 7
    parents = some_parents(B, N, W, g)
    states = [torch.randn(B, N, 1 + i, generator=g).cuda() for i in range(60)]
    for a, b in zip(reorder_states(states, parents), plain_reorder(states, parents)):
        assert torch.equal(a.cpu(), b)
    x = torch.randn(N, B, 40, generator=g).cuda()
    odd = torch.randn(B, 2 * N, 41, generator=g).bfloat16().cuda()
    layered = torch.randn(2, B, N, 24, generator=g).cuda()       # layers first
    shared = torch.randn(1, N, 10, generator=g).cuda().expand(B, N, 10)
    columns = torch.randn(B, N, 5, 6, generator=g).cuda().transpose(2, 3)
    states = [x.transpose(0, 1), odd[:, ::2, 1:], odd[:, 1::2, :40], layered[0], layered[1], shared, columns]
    for a, b in zip(reorder_states(states, parents), plain_reorder(states, parents)):
        assert torch.equal(a.cpu(), b)
    out = [torch.ones(W, B, 40).cuda().transpose(0, 1), torch.ones(B, W, 50).bfloat16().cuda()[:, :, 3:43],
           torch.ones(B, 2 * W, 40).bfloat16().cuda()[:, ::2]]
    want = plain_reorder(states[:3], parents, out)
    reorder_states(states[:3], parents, out=out)
    for a, b in zip(out, want):
        assert torch.equal(a.cpu(), b)


def test_large_states():
    g = torch.Generator().manual_seed(5)
    s = torch.randint(0, 255, (2, 3, 200, 5001), generator=g).to(torch.uint8).cuda()
    parents = torch.tensor([[2, 2, 0, 1], [1, -1, 1, 0]], dtype=torch.int32).cuda()
    got = reorder_states(s, parents)
    assert torch.equal(got[0], s[0, [2, 2, 0, 1]]) and torch.equal(got[1, [0, 2, 3]], s[1, [1, 1, 0]])
    assert not got[1, 1].any()
    want = plain_reorder([s], parents[:, :3].contiguous(), [s])[0]
    reorder_states(s, parents[:, :3].contiguous(), out=s)
    assert torch.equal(s.cpu(), want)


def test_states_beyond_32_bit_offsets():
    s = torch.zeros(1, 5, 2 ** 30, dtype=torch.uint8, device="cuda")
    s[0, :, -1] = torch.arange(1, 6, device="cuda")
    s[0, :, 12345] = torch.arange(11, 16, device="cuda")
    parents = torch.tensor([[4, 3, 4]], dtype=torch.int32).cuda()
    got = reorder_states(s, parents)
    assert got[0, :, -1].tolist() == [5, 4, 5] and got[0, :, 12345].tolist() == [15, 14, 15]
    parents = torch.tensor([[4, 0, 4, 1, 3]], dtype=torch.int32).cuda()
    reorder_states(s, parents, out=s)
    assert s[0, :, -1].tolist() == [5, 1, 5, 2, 4] and s[0, :, 12345].tolist() == [15, 11, 15, 12, 14]


def test_parents_beyond():
    s = torch.arange(6.0).view(1, 3, 2).cuda()
    parents = torch.tensor([[0, 3]], dtype=torch.int32).cuda()
    with pytest.raises(ValueError, match="Parent index mismatch"):
        reorder_states(s, parents)
    assert reorder_states(s, parents, validate_parents=False).tolist() == [[[0.0, 1.0], [0.0, 0.0]]]
    with pytest.raises(ValueError, match="Parent index mismatch"):
        reorder_states([s[..., :0]], parents)
    with pytest.raises(ValueError, match="Parent index mismatch"):
        reorder_states(s, parents, out=s[:, :2])
    assert reorder_states(s, parents[:, :0]).shape == (1, 0, 2)
    assert not reorder_states(s[:, :0], torch.full((1, 2), -1, dtype=torch.int32).cuda()).any()


def test_states_in_a_graph():
    g = torch.Generator().manual_seed(6)
    states, parents = some_states(3, 5, g), some_parents(3, 5, 5, g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        reorder_states(states, parents, out=states, validate_parents=False)
    for _ in range(3):
        parents.copy_(some_parents(3, 5, 5, g))
        want = plain_reorder(states, parents, states)
        graph.replay()
        assert all(torch.equal(a.cpu(), b) for a, b in zip(states, want))


# ---- embeddings -------------------------------------------------------------------------------

def table_and_words(R, H, shape, dtype=torch.float32, seed=0, none=0.1, skew=3.0):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(R, H, generator=g).to(dtype).cuda()
    words = (torch.rand(shape, generator=g) ** skew * R).int().clamp(max=R - 1)
    words[torch.rand(shape, generator=g) < none] = -1
    deltas = torch.randn(*shape, H, generator=g).to(dtype).cuda()
    return table, words.cuda(), deltas


def check_rows(rows, table, words, scale, dropout, seed):
    """One product with a factor that is rounded itself, and one rounding to the type."""
    want, here = ref.embed(table, words, scale, dropout, seed)
    got = rows.detach().cpu().double().flatten(0, -2)
    assert rows.shape == (*words.shape, table.shape[1]) and rows.dtype == table.dtype
    error = 2.02 * UNIT + (half_step(rows.dtype) * 1.01 if rows.dtype is torch.bfloat16 else 0.0)
    assert ((got - want).abs() <= error * want.abs() + 1e-38).all()
    assert (got[~here] == 0).all()
    return here


def check_grad(grad, R, words, deltas, here, scale, dropout):
    """count - 1 additions, the factor and its product in 32 bits, and one rounding to the type."""
    want, size, count = ref.embed_grad(R, words, deltas, here, scale, dropout)
    got = grad.cpu().double()
    bound = (count + 2) * UNIT * 1.01 * size + 1e-38
    if grad.dtype is torch.bfloat16:
        bound = bound + 1.01 * half_step(grad.dtype) * (want.abs() + bound)
    assert grad.shape == (R, deltas.shape[-1])
    assert ((got - want).abs() <= bound).all()


def check_embed(R, H, shape, dtype, scale=1.0, dropout=0.0, seed=None, **options):
    table, words, deltas = table_and_words(R, H, shape, dtype, **options)
    table.requires_grad_(True)
    rows = embed_words(table, words, scale=scale, dropout=dropout, seed=seed)
    here = check_rows(rows, table, words, scale, dropout, 0 if seed is None else int(seed))
    grad, = torch.autograd.grad(rows, table, deltas)
    check_grad(grad, R, words, deltas, here, scale, dropout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,H,shape", [
    (1, 1, (1,)), (1, 8, (3, 2)), (5, 3, (2, 11)), (30, 128, (2, 11)), (28, 17, (1, 1)), (7, 33, (300,)),
    (257, 40, (4, 100)), (1000, 64, (3, 4, 5)), (149, 1025, (16, 21)), (296, 641, (64,)), (3000, 256, (50, 41)),
    (40000, 24, (10, 100)), (70000, 8, (63,)), (2, 264, (1000,)), (300, 2056, (32, 4))])
def test_embeddings(R, H, shape, dtype):
    check_embed(R, H, shape, dtype)
    check_embed(R, H, shape, dtype, scale=H ** 0.5, dropout=0.3, seed=2 ** 40 + 77)


@pytest.mark.parametrize("count", [63, 64, 65, 127, 128, 1000, 4096, 30011])
def test_frequent_words(count):
    """One word almost throughout: its sum is made in parts."""
    for dtype in TYPES:
        check_embed(3, 40, (count,), dtype, none=0.0, skew=20.0, seed=None)
        check_embed(500, 13, (count,), dtype, none=0.02, skew=9.0, dropout=0.5, seed=-3)
    table, words, deltas = table_and_words(4, 16, (count,))
    words[:] = 2
    rows = embed_words(table.requires_grad_(True), words)
    grad, = torch.autograd.grad(rows, table, deltas)
    check_grad(grad, 4, words, deltas, torch.ones(count, 16, dtype=torch.bool), 1.0, 0.0)


@pytest.mark.parametrize("dropout", [1e-9, 1e-5, 0.1, 0.5, 0.99999, 1.0 - 1e-9])
def test_shares(dropout):
    check_embed(20, 50, (40,), torch.float32, dropout=dropout, seed=5)


def test_no_words_and_none_that_count():
    for dtype in TYPES:
        table, words, _ = table_and_words(6, 12, (2, 4), dtype)
        table.requires_grad_(True)
        rows = embed_words(table, words[:, :0])
        grad, = torch.autograd.grad(rows, table, torch.zeros(2, 0, 12, dtype=dtype, device="cuda"))
        assert rows.shape == (2, 0, 12) and grad.shape == (6, 12) and not grad.any()
        rows = embed_words(table, torch.full_like(words, -1))
        grad, = torch.autograd.grad(rows, table, torch.ones_like(rows))
        assert not rows.any() and not grad.any()
        assert embed_words(table[:0], torch.full_like(words, -1)).shape == (2, 4, 12)
        assert embed_words(table[:, :0], words).shape == (2, 4, 0)


def test_scalar_word():
    table, _, _ = table_and_words(6, 12, (1,))
    row = embed_words(table, torch.tensor(3, dtype=torch.int32).cuda(), scale=2.0)
    assert torch.equal(row, 2.0 * table[3])


def test_words_beyond():
    table, words, _ = table_and_words(6, 12, (2, 4))
    words[1, 1], words[0, 2] = 6, 2 ** 31 - 1
    with pytest.raises(ValueError, match="Word index mismatch"):
        embed_words(table, words)
    with pytest.raises(ValueError, match="Word index mismatch"):
        embed_words(table[:, :0], words)
    with pytest.raises(ValueError, match="Word index mismatch"):
        embed_words(table.detach().requires_grad_(True), words)
    words[0, 3] = -2 ** 31
    rows = embed_words(table.requires_grad_(True), words, validate_words=False)
    grad, = torch.autograd.grad(rows.sum(), table)
    here = check_rows(rows, table, words, 1.0, 0.0, 0)
    check_grad(grad, 6, words, torch.ones_like(rows), here, 1.0, 0.0)


def test_numbers_that_are_none_stay_where_they_are():
    """Infinities and NaN in rows that no word has, and in places that are dropped."""
    R, H = 5, 64
    table, words, deltas = table_and_words(R, H, (30,), none=0.0)
    _, here = ref.embed(table, words, 1.0, 0.5, 9)
    table[4] = math.nan
    words[words == 4] = 3
    deltas[~here.cuda()] = math.inf
    rows = embed_words(table.requires_grad_(True), words, dropout=0.5, seed=9)
    grad, = torch.autograd.grad(rows, table, deltas)
    assert rows.isfinite().all() and grad.isfinite().all()
    check_grad(grad, R, words, torch.where(here.cuda(), deltas, 0.0), here, 1.0, 0.5)


def test_strides_of_tables_and_gradients():
    table, words, deltas = table_and_words(50, 24, (6, 7))
    want = embed_words(table, words, scale=3.0)
    wide = torch.zeros(100, 40, device="cuda")
    views = [wide[::2, 8:32].copy_(table), wide[1::2, 5:29].copy_(table), table.t().contiguous().t(),
             torch.zeros(60, 24, device="cuda")[10:].copy_(table)]
    for view in views:
        view = view.detach().requires_grad_(True)
        rows = embed_words(view, words, scale=3.0)
        assert torch.equal(rows, want)
        for d in (deltas, deltas.transpose(0, 1).contiguous().transpose(0, 1), deltas[:1, :1, :1].expand_as(deltas)):
            grad, = torch.autograd.grad(rows, view, d, retain_graph=True)
            check_grad(grad, 50, words, d, ref.embed(table, words)[1], 3.0, 0.0)
    shared = torch.randn(24, device="cuda").expand(50, 24).requires_grad_(True)
    assert torch.equal(embed_words(shared, words)[words >= 0][0], shared[0])


def test_gradient_against_differences():
    """The rows are linear in the table: a difference is the gradient, to the rows' roundings."""
    table, words, deltas = table_and_words(9, 20, (3, 5))
    table.requires_grad_(True)
    grad, = torch.autograd.grad(embed_words(table, words, 2.0, 0.4, 11), table, deltas)
    g = torch.Generator().manual_seed(1)
    for _ in range(5):
        step = torch.randn(9, 20, generator=g).cuda()
        up, down = (embed_words(table.detach() + s * step, words, 2.0, 0.4, 11).double() for s in (1, -1))
        slope = ((up - down) / 2 * deltas.double()).sum().item()
        # (a row is off by four roundings of numbers below 2 / 0.6 * 8)
        assert abs(slope - (grad.double() * step.double()).sum().item()) <= 300 * 8 * 27 * 4 * UNIT


def test_seeds():
    """A number, or one on the device: the same rows, in the forward and in the backward call; graphs see new ones."""
    table, words, deltas = table_and_words(40, 100, (4, 9))
    table.requires_grad_(True)
    rows = embed_words(table, words, dropout=0.25, seed=-12345678901)
    place = torch.tensor([-12345678901]).cuda()
    again = embed_words(table, words, dropout=0.25, seed=place)
    assert torch.equal(rows, again)
    grads = [torch.autograd.grad(r, table, deltas, retain_graph=True)[0] for r in (rows, again)]
    assert torch.equal(*grads)
    assert not torch.equal(rows, embed_words(table, words, dropout=0.25, seed=-12345678900))
    place += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(again, table, deltas)
    leaf = table.detach().clone().requires_grad_(True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = embed_words(leaf, words, dropout=0.25, seed=place, validate_words=False)
        grad, = torch.autograd.grad(held, leaf, deltas)
    for seed in (3, 2 ** 50, -1):
        place.fill_(seed)
        graph.replay()
        here = check_rows(held, leaf, words, 1.0, 0.25, seed)
        check_grad(grad, 40, words, deltas, here, 1.0, 0.25)


def test_embeddings_are_the_same_from_run_to_run():
    table, words, deltas = table_and_words(200, 72, (5000,), skew=4.0)
    table.requires_grad_(True)
    first = None
    for _ in range(4):
        rows = embed_words(table, words, dropout=0.1, seed=4)
        grad, = torch.autograd.grad(rows, table, deltas)
        first = first or (rows, grad)
        assert torch.equal(rows, first[0]) and torch.equal(grad, first[1])


def test_second_derivatives_are_refused():
    table, words, deltas = table_and_words(6, 12, (2, 4))
    table.requires_grad_(True)
    deltas.requires_grad_(True)
    grad, = torch.autograd.grad(embed_words(table, words), table, deltas, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once only"):
        grad.sum().backward()


def test_words_that_change_before_the_backward_call():
    table, words, deltas = table_and_words(6, 12, (2, 4))
    rows = embed_words(table.requires_grad_(True), words)
    words += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(rows, table, deltas)


# ---- together ---------------------------------------------------------------------------------

def test_training_a_table_of_predictions():
    """Predictions that depend on the word before: rows of a table, trained with the loss."""
    from oracle import oracle as O
    B, T, U, V = 3, 20, 6, 30
    g = torch.Generator().manual_seed(2)
    E = torch.randn(B, T, V, generator=g).cuda().requires_grad_(True)
    table = torch.randn(V, V, generator=g).cuda().requires_grad_(True)
    labels = torch.randint(1, V, (B, U), generator=g).int().cuda()
    in_lens, lab_lens = torch.tensor([20, 15, 9]).int().cuda(), torch.tensor([6, 2, 0]).int().cuda()
    n = torch.arange(U + 1, device="cuda")
    words = torch.nn.functional.pad(labels, (1, 0)).masked_fill(n > lab_lens[:, None], -1)
    P = embed_words(table, words)
    costs = TransducerLoss(blank=0)(E, P, labels, in_lens, lab_lens)
    egrad, tgrad = torch.autograd.grad(costs.sum(), (E, table))
    host = [x.detach().cpu().numpy() for x in (E, P, labels, in_lens, lab_lens)]
    want = O.loss_and_grads(*host, blank=0)
    assert torch.allclose(costs.cpu(), torch.from_numpy(want["costs"]), rtol=1e-4)
    sums = torch.zeros(V, V).index_add_(0, words.clamp(min=0).flatten().long().cpu(),
                                        torch.from_numpy(want["pgrads"]).flatten(0, 1))
    assert (tgrad.cpu() - sums).abs().max() <= 1e-3 * sums.abs().max()


def test_a_search():
    """Frame by frame, at most one label each: the words, states and scores of a search on the CPU in 64 bits."""
    B, T, V, H, W = 3, 12, 50, 24, 4
    g = torch.Generator().manual_seed(3)
    E = (2.0 * torch.randn(B, T, V, generator=g)).cuda()
    table = torch.randn(V, H, generator=g).cuda()
    out = (torch.randn(H, V, generator=g) / H ** 0.5).cuda()
    lens = [12, 7, 1]

    scores = torch.full((B, W), -INF).cuda()
    scores[:, 0] = 0.0
    state = torch.zeros(B, W, H).cuda()                      # the predictor: a running mean of embeddings
    history = torch.full((B, W, T), -1, dtype=torch.int32).cuda()
    positions = torch.arange(W, dtype=torch.int32).cuda().repeat(B, 1)
    beams = [[(0.0, [], torch.zeros(H))] for _ in range(B)]
    for t in range(T):
        frames = torch.tensor([[t if t < n else -1] * W for n in lens], dtype=torch.int32).cuda()
        P = state @ out
        scores, parents, words = extend_beams(E, P, frames, positions, scores, W, validate_nodes=False)
        state, history = reorder_states([state, history], parents, validate_parents=False)
        label = words > 0
        history[:, :, t] = torch.where(label, words, -1)
        fresh = embed_words(table, torch.where(label, words, -1), scale=0.5, validate_words=False)
        state = torch.where(label[..., None], 0.5 * state + fresh, state)
        for b in range(B):
            if t >= lens[b]:
                continue
            all_ = []
            for s, said, h in beams[b]:
                z = E[b, t].cpu() + (h @ out.cpu())
                log_p = torch.log_softmax(z.double(), 0)
                for v in range(V):
                    nh = 0.5 * h + 0.5 * table[v].cpu() if v else h
                    all_.append((s + log_p[v].item(), said + [v] if v else said, nh))
            all_.sort(key=lambda x: -x[0])
            assert all_[W - 1][0] - all_[W][0] > 1e-4        # (the search is not on the edge)
            beams[b] = all_[:W]
    for b in range(B):
        for w, (s, said, h) in enumerate(beams[b]):
            assert [x for x in history[b, w].tolist() if x > 0] == said
            assert abs(scores[b, w].item() - s) <= 1e-4
            assert (state[b, w].cpu() - h).abs().max() <= 1e-4
