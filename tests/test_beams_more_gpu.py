"""reorder_states, extend_beams and embed_words on a GPU: calls beside those of test_beams_gpu.py."""
import pytest
import torch

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
