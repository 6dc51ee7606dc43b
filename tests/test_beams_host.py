"""CPU tests of what reorder_states and embed_words hand to the native calls: these are replaced by plain ones on host
memory, so that addresses and lifetimes are looked at where a wrong one harms nothing."""
import ctypes

import pytest
import torch

from transducer_b200 import beams, reorder_states


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
