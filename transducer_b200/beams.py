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
from .nodes import (MAX_LISTED_WORDS, OnDevice, _describe, _rows, certify_nodes, check_device, check_no_tangents)
from .torch_binding import check_contiguous, check_dim, check_type

MAX_REORDERED_WIDTH = 4096


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
    ``validate_nodes=False`` skips the check that no node of a hypothesis lies beyond its tensor (an index that does
    is taken for none), which waits for the kernels, so that the call only enqueues work."""
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
    if scores.is_neg():
        scores = scores.resolve_neg()
    B, N = frames.shape
    device = emissions.device
    with OnDevice(device):
        best = scores.new_empty((B, width))
        parents = frames.new_empty((B, width))
        words = torch.empty_like(parents)
        described, sizes = _describe(emissions, predictions, frames)
        nbytes = _transducer.extend_beams_workspace_bytes(B, sizes[3], N)
        ws = frames.new_empty((nbytes + 3) // 4)
        beyond = _transducer.extend_beams(described, frames.data_ptr(), positions.data_ptr(), scores.data_ptr(),
                                          best.data_ptr(), parents.data_ptr(), words.data_ptr(), sizes, width,
                                          validate_nodes, ws.data_ptr(), nbytes)
    if beyond:
        raise ValueError("Frame index mismatch" if beyond & 1 else "Position index mismatch")
    return best, parents, words


def reorder_states(states, parents, out=None, validate_parents=True):
    """What belongs to hypotheses, for those that follow them: ``states[b, parents[b, w]]`` for every w.

    ``states``   a tensor [B, N, ...] of any type, or a list or tuple of them (predictor states, words so
                 far, keys and values); what follows the second dimension has to be contiguous, and nothing
                 lazily conjugated or negated, or is copied
    ``parents``  int32 [B, W], as from `extend_beams`: a negative one says that there is no hypothesis
    ``out``      tensors [B, W, ...] to write, else they are made; any of them may be its state itself (or
                 its first W hypotheses), which is then reordered in place (at most 4096 hypotheses).  It
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
    device = parents.device
    N = -1
    for s in states:
        shape = s.shape
        if len(shape) < 2:
            raise ValueError("states must have a dimension of utterances and one of hypotheses.")
        if shape[0] != B:
            raise ValueError("must have states per example.")
        if N >= 0 and shape[1] != N:
            raise ValueError("states must have the same number of hypotheses.")
        N = shape[1]
        if s.device != device:
            raise ValueError("all inputs must be on the same device.")
    check_no_tangents(*states)
    if out is not None:
        _check_outputs(states, out, parents)
    with OnDevice(device):
        made = out is None
        if made:
            out = []
        rows, moved = [], []
        copies = []   # (which have to live until the kernels are enqueued: `moved` has addresses)
        for i, s in enumerate(states):
            if (s.is_conj() or s.is_neg()) and (made or not _alike(s, out[i])):
                s = s.detach().resolve_conj().resolve_neg()
                copies.append(s)
            row = _row(s)
            if row is None:
                s = s.detach().contiguous()
                copies.append(s)
                row = _row(s)
            at, from_b, from_n, size = row
            if made:
                o = torch.empty_like(s) if W == N and s.is_contiguous() else s.new_empty((B, W) + s.shape[2:])
                out.append(o)
                moved += at, o.data_ptr(), from_b, from_n, W * size, size, size
            else:
                to, to_b, to_n, _ = _row(out[i])
                rows.append(row)
                moved += at, to, from_b, from_n, to_b, to_n, size
        if not made:
            _check_apart(rows, out, B, N, W, parents)
        beyond = 0
        if B * W:
            beyond = _transducer.reorder_states(moved, parents.data_ptr(), B, N, W, not made, validate_parents)
            if not made:   # (written behind autograd's back)
                torch.autograd.graph.increment_version([o for o in out if not o.is_inference()])
    if beyond:
        raise ValueError("Parent index mismatch")
    return out[0] if single else list(out)


def _check_outputs(states, out, parents):
    if len(out) != len(states):
        raise ValueError("must have an output per state.")
    for s, o in zip(states, out):
        if o.dtype != s.dtype:
            raise TypeError("out must have the states' types")
        if o.shape[:2] != parents.shape or o.shape[2:] != s.shape[2:]:
            raise ValueError("out must have the shape of the reordered states.")
        if _row(o) is None:
            raise ValueError("out must be contiguous behind its second dimension")
        if o.requires_grad:
            raise ValueError("out must not require gradients")
        if (o.is_conj() or o.is_neg()) and not _alike(s, o):
            raise ValueError("out must not be lazily conjugated or negated where its state is not")
    check_device(parents, *out)


def _alike(s, o):
    """Whether the same bytes are the same numbers: tensors may be conjugated or negated when they are read."""
    return s.is_conj() == o.is_conj() and s.is_neg() == o.is_neg()


def _row(s):
    """Where a tensor begins, its bytes from one utterance and from one hypothesis to the next, and bytes of a row; None
    where a hypothesis' numbers are not next to each other."""
    shape = s.shape
    if s.is_contiguous() and shape[0] * shape[1]:
        size = s.nbytes // (shape[0] * shape[1])
        return s.data_ptr(), shape[1] * size, size, size
    stride, size = s.stride(), s.element_size()
    numbers = 1
    for i in range(len(shape) - 1, 1, -1):
        n = shape[i]
        if n != 1 and stride[i] != numbers and s.numel():
            return None
        numbers *= n
    return s.data_ptr(), stride[0] * size, stride[1] * size, numbers * size


def _end(row, B, N):
    """The address behind a tensor of B utterances and N hypotheses; its beginning if it is empty."""
    return row[0] + ((B - 1) * row[1] + (N - 1) * row[2] + row[3] if B * N * row[3] else 0)


def _shared(row, B, N):
    """Whether rows of a tensor of B utterances and N hypotheses share memory."""
    _, by_b, by_n, size = row
    if by_b >= by_n * (N - 1) + size and by_n >= size:   # (one utterance behind the other)
        return False
    for n in range(N):   # rows n hypotheses and b utterances apart begin b * by_b + n * by_n bytes apart
        if by_b == 0:
            least, most = (1 - B, B - 1) if n * by_n < size else (1, 0)
        else:
            least, most = max(1 - B, -((size - 1 + n * by_n) // by_b)), min(B - 1, (size - 1 - n * by_n) // by_b)
        if least <= most and (n > 0 or most > 0):
            return True
    return False


def _check_apart(rows, out, B, N, W, parents):
    """That outputs overlap with nothing, but for one that is its state itself (the same place for every hypothesis)."""
    taken = [(parents.data_ptr(), parents.data_ptr() + parents.nbytes)]
    ends = [_end(row, B, N) for row in rows]
    for i, o in enumerate(out):
        mine = _row(o)
        begin, end = mine[0], _end(mine, B, W)
        if begin == end:
            continue
        reach = mine[3]
        for step, n in sorted(((mine[1], B), (mine[2], W))):   # rows of `o` that share memory
            if n > 1 and step < reach:
                raise ValueError("out must not overlap with itself")
            reach += step * (n - 1)
        for j, row in enumerate(rows):
            if end <= row[0] or ends[j] <= begin:
                continue
            if i != j or begin != row[0] or (B > 1 and mine[1] != row[1]) or (min(N, W) > 1 and mine[2] != row[2]):
                raise ValueError("out must be a state itself or not overlap with the states")
            if W > MAX_REORDERED_WIDTH:
                raise ValueError("at most %d hypotheses are reordered in place" % MAX_REORDERED_WIDTH)
            if N > W and _shared(row, B, N):
                raise ValueError("rows of a state that is reordered in place must not be another utterance's")
        for other in taken:
            if begin < other[1] and other[0] < end:
                raise ValueError("outputs must not overlap with each other or with parents")
        taken.append((begin, end))
