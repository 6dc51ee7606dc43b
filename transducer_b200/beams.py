"""A beam search's step: the best extensions of every utterance's hypotheses (`extend_beams`) and the
states that follow them (`reorder_states`).  The reference decodes given transcripts only and has neither.

Hypotheses are at nodes of the lattice, see `transducer_b200.nodes`: hypothesis n of utterance b is at
frame ``frames[b, n]`` and label position ``positions[b, n]``, a row of its own in ``predictions`` or one
that it shares (a predictor that looks at the last word alone is a table of such rows:
``predictions=table.expand(B, -1, -1)``, with the last words as positions).  A step extends every
hypothesis by the blank (to the next frame) or a label (to the next position); the caller moves the
nodes, which frame a word leads to is no concern of these functions.

CUDA tensors only, like `TransducerLoss`; the work is enqueued on torch's current stream."""
import torch

from . import _transducer
from .nodes import (MAX_LISTED_WORDS, OnDevice, _describe, _rows, certify_indices, certify_nodes, check_device,
                    check_no_tangents)
from .torch_binding import check_contiguous, check_dim, check_type

MAX_REORDERED_WIDTH = 8192


def extend_beams(emissions, predictions, frames, positions, scores, width, validate_nodes=True):
    """The ``width`` best extensions of each utterance's hypotheses (at most 256).

    ``scores`` float32 [B, N] are the hypotheses' log-probabilities; one of -inf says that there is no
    hypothesis (its node is not looked at), one without a node (a negative index) that it is finished: it
    competes as it is, with word -1.  Word v, the blank like any other, extends hypothesis n to the score
    ``scores[b, n] + log_softmax(z)[v]``.

    Returns scores float32, parents int32 and words int32, all [B, width]: the greatest score first, of
    equal ones the lower parent, then the lower word; -inf, -1, -1 where there are fewer (words whose z is
    -inf are none).  The order is that of 64-bit arithmetic.  An utterance with a hypothesis whose score is
    NaN or +inf, or that has such a z, gets NaN, -1, -1.  The results are detached from the inputs' graph.
    ``validate_nodes``: see `top_words`; an index beyond its tensor is taken for no node."""
    certify_nodes(emissions, predictions, frames, positions)
    check_no_tangents(emissions, predictions, scores)
    check_dim(scores, 2, "scores")
    check_type(scores, torch.float32, "scores")
    check_contiguous(scores, "scores")
    if scores.shape != frames.shape:
        raise ValueError("must have a score per node.")
    check_device(emissions, scores)
    if not 1 <= width <= MAX_LISTED_WORDS:
        raise ValueError("width must be between 1 and %d" % MAX_LISTED_WORDS)
    emissions, predictions = _rows(emissions), _rows(predictions)
    B, N = frames.shape
    device = emissions.device
    with OnDevice(device):
        best = torch.empty((B, width), device=device, dtype=torch.float32)
        parents = torch.empty((B, width), device=device, dtype=torch.int32)
        words = torch.empty((B, width), device=device, dtype=torch.int32)
        described, sizes = _describe(emissions, predictions, frames)
        nbytes = _transducer.extend_beams_workspace_bytes(B, sizes[3], N)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _transducer.extend_beams(described, frames.data_ptr(), positions.data_ptr(), scores.data_ptr(),
                                 best.data_ptr(), parents.data_ptr(), words.data_ptr(), sizes, width,
                                 ws.data_ptr(), nbytes)
        if validate_nodes:
            certify_indices(emissions, predictions, frames, positions)
    return best, parents, words


def reorder_states(states, parents, out=None, validate_parents=True):
    """What belongs to hypotheses, for those that follow them: ``states[b, parents[b, w]]`` for every w.

    ``states``   a tensor [B, N, ...] of any type, or a list or tuple of them (predictor states, words so
                 far, keys and values); what follows the second dimension has to be contiguous, or is copied
    ``parents``  int32 [B, W], as from `extend_beams`: a negative one says that there is no hypothesis
    ``out``      tensors [B, W, ...] to write, else they are made; any of them may be its state itself (or
                 its first W hypotheses), which is then reordered in place (at most 8192 hypotheses).  It
                 must not overlap with others.

    Returns the new states as they came: a tensor, or a list.  Rows without a hypothesis are left as they were
    in ``out``, and zeros in tensors that are made here.  The results are detached from the states' graph.
    ``validate_parents=False`` skips the check that no parent is N or more (such ones are taken for none),
    which waits for the kernels, so that the call only enqueues work."""
    check_dim(parents, 2, "parents")
    check_type(parents, torch.int32, "parents")
    check_contiguous(parents, "parents")
    single = isinstance(states, torch.Tensor)
    if single:
        states, out = [states], None if out is None else [out]
    if not len(states):
        raise ValueError("there must be a state to reorder.")
    B, W = parents.shape
    N = states[0].shape[1] if states[0].dim() >= 2 else 0
    for s in states:
        if s.dim() < 2:
            raise ValueError("states must have a dimension of utterances and one of hypotheses.")
        if s.shape[0] != B:
            raise ValueError("must have states per example.")
        if s.shape[1] != N:
            raise ValueError("states must have the same number of hypotheses.")
    check_device(parents, *states)
    check_no_tangents(*states)
    if out is not None:
        if len(out) != len(states):
            raise ValueError("must have an output per state.")
        for s, o in zip(states, out):
            if o.dtype != s.dtype:
                raise TypeError("out must have the states' types")
            if tuple(o.shape) != (B, W) + tuple(s.shape[2:]):
                raise ValueError("out must have the shape of the reordered states.")
            if not _together(o):
                raise ValueError("out must be contiguous behind its second dimension")
            if o.requires_grad:
                raise ValueError("out must not require gradients")
        check_device(parents, *out)
    with OnDevice(parents.device):
        kept = out is not None
        states = [s if _together(s) else s.detach().contiguous() for s in states]
        if kept:
            _check_apart(states, out, W)
        else:
            out = [s.new_empty((B, W) + tuple(s.shape[2:])) for s in states]
        if B * W:
            _transducer.reorder_states([_moved(s, o) for s, o in zip(states, out)], parents.data_ptr(), B, N, W,
                                       kept)
            if kept:   # (written behind autograd's back)
                torch.autograd.graph.increment_version([o for o in out if not o.is_inference()])
            if validate_parents:
                certify_parents(parents, N)
    return out[0] if single else list(out)


def certify_parents(parents, N):
    """That no parent lies beyond the N hypotheses; see nodes.certify_indices."""
    scratch = torch.empty(_transducer.node_summary_scratch_bytes, dtype=torch.uint8, device=parents.device)
    most = _transducer.node_summary(0, 0, 0, parents.data_ptr(), parents.numel(), scratch.data_ptr())[2]
    if most >= N:
        raise ValueError("Parent index mismatch")


def _row_numbers(s):
    n = 1
    for size in s.shape[2:]:
        n *= size
    return n


def _together(s):
    """Whether a hypothesis' numbers are next to each other."""
    want = 1
    for size, stride in zip(reversed(s.shape[2:]), reversed(s.stride()[2:])):
        if size != 1 and stride != want:
            return _row_numbers(s) == 0
        want *= size
    return True


def _moved(s, o):
    size = s.element_size()
    (sb, sn), (ob, on) = s.stride()[:2], o.stride()[:2]
    return s.data_ptr(), o.data_ptr(), sb * size, sn * size, ob * size, on * size, _row_numbers(s) * size


def _extent(s):
    """Addresses from the first byte to behind the last one; None if there are none."""
    if s.numel() == 0:
        return None
    last = sum((n - 1) * k for n, k in zip(s.shape, s.stride()))
    return s.data_ptr(), s.data_ptr() + (last + 1) * s.element_size()


def _check_apart(states, out, W):
    taken = []
    for i, o in enumerate(out):
        mine = _extent(o)
        if mine is None:
            continue
        row = _row_numbers(o)
        sizes = sorted((k, n) for n, k in zip(o.shape[:2], o.stride()[:2]) if n > 1)
        reach = row
        for k, n in sizes:   # rows of `o` that share memory
            if k < reach:
                raise ValueError("out must not overlap with itself")
            reach = k * (n - 1) + reach
        for j, s in enumerate(states):
            other = _extent(s)
            if other is None or mine[1] <= other[0] or other[1] <= mine[0]:
                continue
            if i != j or not _same_place(s, o):
                raise ValueError("out must be a state itself or not overlap with the states")
            if W > MAX_REORDERED_WIDTH:
                raise ValueError("at most %d hypotheses are reordered in place" % MAX_REORDERED_WIDTH)
        for other in taken:
            if mine[0] < other[1] and other[0] < mine[1]:
                raise ValueError("outputs must not overlap with each other")
        taken.append(mine)


def _same_place(s, o):
    """Whether hypothesis n of utterance b lies at the same address in both."""
    if s.data_ptr() != o.data_ptr():
        return False
    same_b = s.shape[0] == 1 or s.stride(0) == o.stride(0)
    same_n = min(s.shape[1], o.shape[1]) == 1 or s.stride(1) == o.stride(1)
    return same_b and same_n
