"""reorder_states, extend_beams and embed_words on a GPU: calls beside those of test_beams_gpu.py."""
import numpy as np
import pytest
import torch

import beam_reference as ref
import test_beams_gpu as base
from transducer_b200 import TransducerLoss, embed_words, extend_beams, reorder_states, top_words

pytestmark = pytest.mark.gpu


# ---- states -----------------------------------------------------------------------------------

@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("shape", [(3, 4, 5, 6), (4, 6, 96, 64)])
def test_several_states_that_are_copied(shape, given):
    """Their copies are all there when the kernels run, whatever is made after them."""
    g = torch.Generator().manual_seed(1)
    B, N, H, D = shape
    parents = base.some_parents(B, N, N, g)
    states = [torch.randn(shape, generator=g).cuda().transpose(2, 3) for _ in range(5)]
    states.append(torch.randn(B, N, D, H, generator=g).cuda())
    out = [torch.full((B, N, D, H), float(i)).cuda() for i in range(6)] if given else None
    want = base.plain_reorder(states, parents, out)
    for _ in range(3):   # (the allocator has blocks of this size by then)
        got = reorder_states(states, parents, out=out)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_states_that_are_read_lazily():
    """Conjugated or negated when they are read: the numbers are moved, not the bytes."""
    g = torch.Generator().manual_seed(2)
    z = torch.complex(*torch.randn(2, 3, 5, 7, generator=g)).cuda()
    parents = base.some_parents(3, 5, 5, g)
    states = [z.conj(), z.conj().imag, z.conj().imag[..., 0], z]
    out = [torch.zeros(s.shape, dtype=s.dtype, device="cuda") for s in states]
    want = base.plain_reorder(states, parents)
    for got in reorder_states(states, parents), reorder_states(states, parents, out=out):
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    want = base.plain_reorder([z.conj()], parents, [z])[0]
    assert torch.equal(reorder_states(z.conj(), parents, out=z).cpu(), want)


# ---- embeddings -------------------------------------------------------------------------------

@pytest.mark.parametrize("how", ["host", "hooks", "checkpoint"])
@pytest.mark.parametrize("shape", [(4, 9), (70, 80)])
def test_seeds_that_the_call_does_not_keep(how, shape):
    """Saved tensors moved to the host, copied by hooks, or made again: the gradient has the rows' own mask."""
    from torch.utils.checkpoint import checkpoint
    seed = 2 ** 50 + 3
    table, words, deltas = base.table_and_words(40, 100, shape)
    table.requires_grad_(True)

    def embed(t):
        return embed_words(t, words, dropout=0.25, seed=torch.tensor([seed]).cuda())
    if how == "checkpoint":
        rows = checkpoint(embed, table, use_reentrant=False)
    else:
        with torch.autograd.graph.save_on_cpu() if how == "host" else \
                torch.autograd.graph.saved_tensors_hooks(lambda x: x.clone(), lambda x: x.clone()):
            rows = embed(table)
    others = [torch.tensor([-1]).cuda() for _ in range(200)]   # (in the seed's place)
    grad, = torch.autograd.grad(rows, table, deltas)
    here = base.check_rows(rows, table, words, 1.0, 0.25, seed)
    base.check_grad(grad, 40, words, deltas, here, 1.0, 0.25)
    del others


def test_as_many_words_as_there_may_be():
    """2^31 - 2 of them, with numbers whose sums are exact in 32 bits."""
    N, R = 2 ** 31 - 2, 1000
    torch.cuda.empty_cache()
    words = torch.arange(R, dtype=torch.int32, device="cuda").repeat(N // R + 1)[:N]
    counts = torch.full((R,), N // R, dtype=torch.int64)
    counts[:N % R] += 1
    for part, word in ((slice(0, 40), 9), (slice(N - 40, N), 7)):
        counts -= torch.bincount(words[part].cpu(), minlength=R)
        counts[word] += 40
        words[part] = word
    words[-1] = -1
    counts[7] -= 1
    table = torch.randn(R, 1, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_(True)
    rows = embed_words(table, words)
    for begin in range(0, N, 2 ** 28):
        some = words[begin:min(N, begin + 2 ** 28)]
        want = table.detach()[:, 0].index_select(0, some.clamp(min=0))
        assert torch.equal(rows.detach()[begin:begin + 2 ** 28, 0], want.mul_(some >= 0))
        del some, want
    deltas = torch.ones_like(rows)
    grad, = torch.autograd.grad(rows, table, deltas)
    assert torch.equal(grad[:, 0].cpu().double(), counts.double())
    del rows, deltas, words
    torch.cuda.empty_cache()


# ---- calls that wait --------------------------------------------------------------------------

def checked_calls():
    E, P, frames, positions, scores = base.hypotheses(2, 3, 4, 200, 3, done=0.0, gone=0.0)
    parents = torch.zeros(2, 3, dtype=torch.int32).cuda()
    labels = torch.ones(2, 3, dtype=torch.int32).cuda()
    lens = torch.full((2,), 3, dtype=torch.int32).cuda()
    return {"extend": lambda: extend_beams(E, P, frames, positions, scores, 2),
            "reorder": lambda: reorder_states(scores, parents),
            "embed": lambda: embed_words(E[0], parents),
            "top": lambda: top_words(E, P, frames, positions, 2),
            "loss": lambda: TransducerLoss(blank=0)(E, P, labels, lens, lens)}


@pytest.mark.parametrize("which", ["extend", "reorder", "embed", "top", "loss"])
def test_other_threads_go_on_while_a_call_waits(which):
    """The stream is busy for a while; another thread counts meanwhile, which takes the interpreter's lock."""
    import threading
    import time
    call = checked_calls()[which]
    call()
    a = torch.randn(8192, 8192, device="cuda")
    torch.cuda.synchronize()
    begins, ends = torch.cuda.Event(), []
    called, done = threading.Event(), threading.Event()

    def work():
        b = a
        for _ in range(60):   # (some 20 ms each)
            b = a @ b * 1e-3
        begins.record()
        called.set()
        call()
        ends.append(begins.query())
        done.set()
    thread = threading.Thread(target=work)
    thread.start()
    called.wait()
    counted = 0
    while not done.is_set() and not begins.query():   # (as long as the stream has not come to the call)
        counted += 1
        time.sleep(1e-3)
    thread.join()
    assert ends == [True]   # (it did wait)
    assert counted >= 50


# ---- ways through the kernels that take many words, rows or numbers -------------------------------

@pytest.mark.parametrize("width", [5, 64, 256])
@pytest.mark.parametrize("N,V", [(300, 1200), (257, 2049), (700, 40)])
def test_equal_scores_of_many_hypotheses(N, V, width):
    """More than are held in shared memory, and more words next to each other than there are lists for."""
    E, P, frames, positions, scores = base.hypotheses(2, 3, N, V, N, seed=N, done=0.05, gone=0.05)
    positions[positions >= 0] = torch.arange(N, device="cuda").repeat(2, 1)[positions >= 0].int()
    flat = torch.where(scores == -base.INF, scores, -5.0)
    few = torch.randint(0, 3, E.shape, generator=torch.Generator().manual_seed(1)).float().cuda()
    for e, p, s in ((0 * E, 0 * P, flat), (few, 0 * P, flat), (1e-7 * E, 1e-7 * P, flat), (few, 0 * P, scores),
                    (E, 1e-7 * P, flat)):
        base.check_extend([e, p, frames, positions, s], width)


@pytest.mark.parametrize("dtype", base.TYPES)
@pytest.mark.parametrize("R,H,count,skew", [
    (3, 40, 70001, 20.0),         # most are one word: more of a warp's than are listed
    (500, 9, 100003, 9.0), (40000, 5, 150000, 30.0),
    (2000, 24, 100003, 3.0),      # 32 places to a warp
    (100, 700, 40000, 3.0), (300, 1030, 16000, 1.0)])
def test_many_words(R, H, count, skew, dtype):
    base.check_embed(R, H, (count,), dtype, skew=skew, none=0.05)
    base.check_embed(R, H, (count,), dtype, skew=skew, none=0.0, scale=0.25, dropout=0.1, seed=77)


def test_one_word_throughout():
    count = 80000
    table, words, deltas = base.table_and_words(4, 16, (count,))
    words[:] = 2
    rows = embed_words(table.requires_grad_(True), words)
    grad, = torch.autograd.grad(rows, table, deltas)
    base.check_grad(grad, 4, words, deltas, torch.ones(count, 16, dtype=torch.bool), 1.0, 0.0)


@pytest.mark.parametrize("dropout", [0.0, 0.5])
def test_embeddings_beyond_32_bit_offsets(dropout):
    """More than 2^31 numbers in the table, in the rows and in the gradient."""
    R = N = 66000
    H, seed = 32776, 12345
    g = torch.Generator().manual_seed(8)
    torch.cuda.empty_cache()
    table = torch.zeros(R, H, dtype=torch.bfloat16, device="cuda")
    some = [0, 1, 65535, R - 2, R - 1]
    table[some] = torch.randn(len(some), H, generator=g).bfloat16().cuda()
    words = torch.randint(2, 65535, (N,), generator=g).int().cuda()
    places = [0, 3, 40000, N - 2, N - 1]
    words[places] = torch.tensor([R - 1, 0, R - 2, 65535, R - 1], dtype=torch.int32).cuda()
    rows = embed_words(table.requires_grad_(True), words, dropout=dropout, seed=seed)
    deltas = torch.zeros_like(rows)
    deltas[places] = torch.randn(len(places), H, generator=g).bfloat16().cuda()
    grad, = torch.autograd.grad(rows, table, deltas)
    groups = H // 8
    counter = np.zeros((len(places), groups, 4), np.uint64)
    counter[..., 0] = np.array(places)[:, None]
    counter[..., 2] = np.arange(groups)
    x = ref.philox(counter, (seed, 0))
    halves = np.stack((x & np.uint64(0xffff), x >> np.uint64(16)), -1).reshape(len(places), H)
    stays = torch.from_numpy(halves >= round(dropout * 65536))
    factor = ref.factor(1.0, dropout)
    # (factors are powers of 2: products are exact, and a sum of two is rounded in 32 bits and to the type)
    want = torch.where(stays, table.detach()[words[places].long()].cpu().double() * factor, 0.0)
    assert torch.equal(rows.detach()[places].cpu().double(), want)
    d = torch.where(stays, deltas[places].cpu().double() * factor, 0.0)
    want = torch.stack((d[1], torch.zeros(H, dtype=torch.float64), d[3], d[2], d[0] + d[4]))
    bound = (base.half_step(torch.bfloat16) + base.UNIT) * 1.01 * want.abs() + base.UNIT * (d[0].abs() + d[4].abs())
    assert ((grad[some].cpu().double() - want).abs() <= bound).all()
    rest = torch.ones(R, dtype=torch.bool, device="cuda")
    rest[some] = False
    assert all(not grad[begin:begin + 8192][rest[begin:begin + 8192]].any() for begin in range(0, R, 8192))
    del rows, deltas, grad, table
    torch.cuda.empty_cache()
