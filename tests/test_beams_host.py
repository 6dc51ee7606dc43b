"""CPU tests of what reorder_states and embed_words hand to the native calls: these are replaced by plain ones on host
memory, so that addresses and lifetimes are looked at where a wrong one harms nothing."""
import ctypes

import pytest
import torch

from transducer_b200 import beams, embed_words, embeddings, extend_beams, reorder_states


class Anywhere(object):
    """In the place of OnDevice."""

    def __init__(self, device):
        pass

    def __enter__(self):
        pass

    def __exit__(self, *exc):
        pass


class Mover(object):
    """reorder_states on the host: every source is read before anything is written, after a look at the addresses."""

    def __init__(self):
        self.calls = 0

    def reorder_states(self, moved, parents, B, N, W, kept, validate):
        self.calls += 1
        states = [moved[i:i + 7] for i in range(0, len(moved), 7)]
        ranges = []
        for at, to, from_b, from_n, to_b, to_n, size in states:
            ranges.append((at, at + (B - 1) * from_b + (N - 1) * from_n + size))
            if to != at:   # (not in place)
                ranges.append((to, to + (B - 1) * to_b + (W - 1) * to_n + size))
        ranges.sort()
        assert all(a[1] <= b[0] for a, b in zip(ranges, ranges[1:])), "sources and outputs share memory"
        parents = (ctypes.c_int * (B * W)).from_address(parents)
        writes = []
        for at, to, from_b, from_n, to_b, to_n, size in states:
            for b in range(B):
                for w in range(W):
                    n = parents[b * W + w]
                    if 0 <= n < N:
                        writes.append((to + b * to_b + w * to_n, ctypes.string_at(at + b * from_b + n * from_n, size)))
                    elif not kept:
                        writes.append((to + b * to_b + w * to_n, bytes(size)))
        for to, data in writes:
            ctypes.memmove(to, data, len(data))
        return 0


@pytest.fixture
def mover(monkeypatch):
    mover = Mover()
    monkeypatch.setattr(beams, "_transducer", mover)
    monkeypatch.setattr(beams, "OnDevice", Anywhere)
    return mover


def plain(states, parents, out=None):
    """states[b, parents[b, w]]; rows without a parent as they are in `out`, else zeros."""
    B, W = parents.shape
    result = []
    for i, s in enumerate(states):
        o = torch.zeros((B, W) + s.shape[2:], dtype=s.dtype) if out is None else out[i].clone()
        for b in range(B):
            for w in range(W):
                if parents[b, w] >= 0:
                    o[b, w] = s[b, parents[b, w]]
        result.append(o)
    return result


PARENTS = torch.tensor([[2, -1, 0], [1, 1, 2]], dtype=torch.int32)


def transposed(count, *shape):
    g = torch.Generator().manual_seed(1)
    return [torch.randn(*shape, generator=g).transpose(2, 3) for _ in range(count)]


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("copied", [1, 2, 3, 8])
def test_states_that_are_copied_live_until_the_kernels_are_enqueued(mover, copied, given):
    """Key and value caches of several layers with their last dimensions the other way around, and a state of the same
    size that needs no copy, which takes the place of what was freed."""
    states = transposed(copied, 2, 3, 4, 6) + [torch.randn(2, 3, 6, 4)]
    out = [torch.full((2, 3, 6, 4), 7.0) for _ in states] if given else None
    want = plain(states, PARENTS, out)
    got = reorder_states(states, PARENTS, out=out)
    assert mover.calls == 1
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- the seed of embed_words --------------------------------------------------------------------

class Embedder(object):
    """embed_words and its gradient on the host, with a mask that shows which seed was read: number (n, h) is dropped where
    bit (n + h) mod 64 of the seed is set."""

    @staticmethod
    def _masked(rows, words, seed, seed_at):
        if seed_at:
            seed = ctypes.c_int64.from_address(seed_at).value
        n, h = torch.arange(rows.shape[0])[:, None], torch.arange(rows.shape[1])
        dropped = torch.tensor([(seed >> i) & 1 for i in range(64)], dtype=torch.bool)[(n + h) % 64]
        return torch.where(dropped, 0.0, rows)

    @staticmethod
    def _tensor(address, kind, dtype, *shape):
        count = 1
        for n in shape:
            count *= n
        return torch.frombuffer((kind * count).from_address(address), dtype=dtype).view(shape)

    def embed_words(self, table, bf16, stride, words, count, rows, R, H, scale, dropout, seed, seed_at, validate):
        words = self._tensor(words, ctypes.c_int, torch.int32, count)
        table = self._tensor(table, ctypes.c_float, torch.float32, (R - 1) * stride + H).as_strided((R, H), (stride, 1))
        self._tensor(rows, ctypes.c_float, torch.float32, count, H).copy_(
            self._masked(table[words.long()], words, seed, seed_at))
        return 0

    def embed_backward_workspace_bytes(self, count, R, H):
        return 0

    def embed_backward(self, deltas, bf16, words, count, grad, R, H, scale, dropout, seed, seed_at, ws, nbytes):
        words = self._tensor(words, ctypes.c_int, torch.int32, count)
        deltas = self._tensor(deltas, ctypes.c_float, torch.float32, count, H)
        grad = self._tensor(grad, ctypes.c_float, torch.float32, R, H)
        grad.zero_().index_add_(0, words.long(), self._masked(deltas, words, seed, seed_at))


@pytest.fixture
def embedder(monkeypatch):
    monkeypatch.setattr(embeddings, "_transducer", Embedder())
    monkeypatch.setattr(embeddings, "OnDevice", Anywhere)


def fresh_seed(value):
    return torch.tensor([value], dtype=torch.int64)


def others():
    """Numbers that take the place of a seed that was freed."""
    return [fresh_seed(-1) for _ in range(200)]


def held_to(grad, table, words, rows, deltas):
    """The gradient has the rows' mask (no number of the table is 0)."""
    kept = rows.detach().flatten(0, -2) != 0
    want = torch.zeros_like(table).index_add_(0, words.flatten().long(), deltas.flatten(0, -2) * kept)
    assert 0.2 < kept.float().mean() < 0.8
    assert torch.equal(grad, want)


SEED = 0x5a5a33cc0f1e6978


def embed_case():
    g = torch.Generator().manual_seed(2)
    table = torch.rand(6, 40, generator=g) + 1.0
    words = torch.randint(0, 6, (5, 7), generator=g).int()
    deltas = torch.randint(1, 9, (5, 7, 40), generator=g).float()   # (sums that are exact)
    return table.requires_grad_(True), words, deltas


@pytest.mark.parametrize("copied", [False, True])
def test_seed_that_goes_through_hooks(embedder, copied):
    """Saved tensors that a hook has copied, as when they are moved to the host: the seed itself is gone by then."""
    table, words, deltas = embed_case()
    pack = (lambda x: x.clone()) if copied else (lambda x: x)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda x: x.clone()):
        rows = embed_words(table, words, dropout=0.5, seed=fresh_seed(SEED))
    held = others()
    grad, = torch.autograd.grad(rows, table, deltas)
    held_to(grad, table, words, rows, deltas)
    del held


def test_seed_of_a_recomputed_call(embedder):
    """Checkpointing makes the call again when the gradient is wanted, its seed with it."""
    from torch.utils.checkpoint import checkpoint
    table, words, deltas = embed_case()
    rows = checkpoint(lambda t: embed_words(t, words, dropout=0.5, seed=fresh_seed(SEED)), table, use_reentrant=False)
    held = others()
    grad, = torch.autograd.grad(rows, table, deltas)
    held_to(grad, table, words, rows, deltas)
    del held


def test_seeds_without_hooks(embedder):
    table, words, deltas = embed_case()
    for seed in (SEED, fresh_seed(SEED)):
        rows = embed_words(table, words, dropout=0.5, seed=seed)
        grad, = torch.autograd.grad(rows, table, deltas)
        held_to(grad, table, words, rows, deltas)
    place = fresh_seed(SEED)
    rows = embed_words(table, words, dropout=0.5, seed=place)
    place += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(rows, table, deltas)


def test_saved_words_that_come_back_elsewhere(embedder):
    """A hook that leaves them on another device, or not one after the other."""
    table, words, deltas = embed_case()
    for unpack, kind, message in [(lambda x: x.to("meta"), ValueError, "same device"),
                                  (lambda x: x.t().contiguous().t() if x.dim() == 2 else x, None, None)]:
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
            rows = embed_words(table, words, dropout=0.5, seed=fresh_seed(SEED))
        if kind is None:
            grad, = torch.autograd.grad(rows, table, deltas)
            held_to(grad, table, words, rows, deltas)
        else:
            with pytest.raises(kind, match=message):
                torch.autograd.grad(rows, table, deltas)


# ---- tensors that are conjugated or negated when they are read ----------------------------------

def lazy(kind, *shape):
    z = torch.complex(*torch.randn(2, *shape, generator=torch.Generator().manual_seed(4)))
    return {"conj": z.conj(), "neg": z.conj().imag, "both": torch.complex(z.imag, z.real).conj()._neg_view(),
            "column": z.conj().imag[..., 0], "plain": z}[kind]


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("kind", ["conj", "neg", "both", "column", "plain"])
def test_states_that_are_read_lazily(mover, kind, given):
    states = [lazy(kind, 2, 3, 5) for _ in range(2)]
    out = [torch.full((2, 3) + s.shape[2:], 7.0, dtype=s.dtype) for s in states] if given else None
    want = plain(states, PARENTS, out)
    got = reorder_states(states, PARENTS, out=out)
    assert all(torch.equal(a, b) and not a.is_conj() and not a.is_neg() for a, b in zip(got, want))


def test_lazy_states_in_place_and_as_outputs(mover):
    x = lazy("plain", 2, 3, 5)
    want = plain([x.conj()], PARENTS, [x])[0]
    got = reorder_states(x.conj(), PARENTS, out=x)   # (the same memory, other numbers)
    assert got is x and torch.equal(x, want)
    lazily = lazy("conj", 2, 3, 5)
    want = plain([lazily], PARENTS, [lazily])[0]
    assert torch.equal(reorder_states(lazily, PARENTS, out=lazily), want)   # in place
    with pytest.raises(ValueError, match="lazily"):
        reorder_states(x, PARENTS, out=torch.zeros_like(x).conj())
    with pytest.raises(ValueError, match="lazily"):
        reorder_states(x.real.contiguous(), PARENTS, out=torch.zeros(2, 3, 5)._neg_view())


def negated(*shape):
    """A negative number throughout, from memory that holds a positive one."""
    return torch.complex(torch.ones(shape), torch.full(shape, 3.0)).conj().imag


@pytest.mark.parametrize("R,H", [(1, 1), (4, 1), (4, 5)])
def test_embeddings_that_are_read_lazily(embedder, R, H):
    words = torch.zeros(1, dtype=torch.int32)
    table = negated(R, H)
    assert torch.equal(embed_words(table, words), table[:1])
    table = table.detach().requires_grad_(True)
    rows = embed_words(table, words)
    assert torch.equal(rows, table[:1])
    grad, = torch.autograd.grad(rows, table, negated(1, H))
    assert torch.equal(grad, torch.cat((negated(1, H), torch.zeros(R - 1, H))))


class Extender(object):
    """Reads what extend_beams hands on of one hypothesis at one node."""

    def extend_beams_workspace_bytes(self, B, V, N):
        return 0

    def extend_beams(self, described, frames, positions, scores, *rest):
        e, p = described[:2]
        self.seen = [ctypes.c_float.from_address(x).value for x in (e, p, scores)]
        return 0


def test_scores_that_are_read_lazily(monkeypatch):
    extender = Extender()
    monkeypatch.setattr(beams, "_transducer", extender)
    monkeypatch.setattr(beams, "OnDevice", Anywhere)
    node = torch.zeros(1, 1, dtype=torch.int32)
    extend_beams(negated(1, 1, 1), negated(1, 1, 1), node, node, negated(1, 1), 1)
    assert extender.seen == [-3.0] * 3
    extend_beams(negated(1, 1, 6), negated(1, 1, 6), node, node, negated(1, 1), 1)
    assert extender.seen == [-3.0] * 3


# ---- states in place whose other rows are utterances' of their own ------------------------------

def shared_bytes(row, B, N):
    """Rows that share memory, by looking at each with each."""
    _, by_b, by_n, size = row
    at = sorted(b * by_b + n * by_n for b in range(B) for n in range(N))
    return size > 0 and any(y - x < size for x, y in zip(at, at[1:]))


def test_rows_in_place_that_are_another_utterances():
    """Only the first W hypotheses are written, but all N may be read."""
    room = torch.zeros(400)
    refused = accepted = 0
    for B, N, W in [(2, 4, 2), (3, 4, 1), (2, 3, 3), (4, 7, 2), (1, 5, 2), (2, 2, 4)]:
        parents = torch.zeros(B, W, dtype=torch.int32)
        for by_b in range(0, 41):
            for by_n in (0, 1, 2, 3, 5, 9, 10):
                for size in (1, 2, 5):
                    whole = room.as_strided((B, max(N, W), size), (by_b, by_n, 1))
                    s, out = whole[:, :N], whole[:, :W]
                    try:
                        beams._check_apart([beams._row(s)], [out], B, N, W, parents)
                    except ValueError:
                        refused += 1
                        # (nothing is refused for the rows that are only read, unless they do share memory)
                        try:
                            beams._check_apart([beams._row(out)], [out], B, W, W, parents)
                        except ValueError:
                            continue
                        assert shared_bytes(beams._row(whole), B, max(N, W))
                    else:
                        accepted += 1
                        assert not shared_bytes(beams._row(whole), B, max(N, W))
    assert refused > 100 and accepted > 100


def test_example_of_such_rows(mover):
    s = torch.zeros(30).as_strided((2, 4, 5), (10, 5, 1))
    parents = torch.tensor([[2, 3], [0, 1]], dtype=torch.int32)
    with pytest.raises(ValueError, match="rows of a state"):
        reorder_states(s, parents, out=s[:, :2])
    assert mover.calls == 0
