"""Operators on single nodes of the transducer's lattice: the best words of a node (`top_words`), a
word drawn from its distribution (`sample_words`) and distillation from a teacher's recorded best
words (`NodeDistillationLoss`).  The reference works on whole lattices only and has none of them.

Node n of utterance b is frame ``frames[b, n]`` and label position ``positions[b, n]`` (both int32
[B, N], in any order, the same node more than once if need be); a negative one says that there is
no node.  Its scores are ``emissions[b, frame, :] + predictions[b, position, :]``, added in 32 bits
(`TransducerLoss` takes the softmax of the same sum).  Words are masked by -inf or any low number.

    emissions    float32 [B, T, V], or both bfloat16; any strides (the words of a row are made
    predictions  float32 [B, U, V]  adjacent if they are not)

The nodes of an alignment are one per blank and label: with its moves, labels being 1, the nodes
that they leave from have positions ``moves.cumsum(1) - moves`` and frames ``arange(N) - positions``.
They are a path (neither frames nor positions go back), which is what the gradients are fastest for;
more than 64 places without a node before another one of the utterance make it none.  A decoder that
extends one hypothesis per utterance passes its frames [B, 1], positions of 0 and predictions [B, 1, V].

CUDA tensors only, like `TransducerLoss`; the work is enqueued on torch's current stream."""
import torch
from torch.autograd import forward_ad

from . import _transducer
from .torch_binding import _workspace, check_contiguous, check_dim, check_type

MAX_LISTED_WORDS = 256


def certify_nodes(emissions, predictions, frames, positions):
    """Argument checks, in the manner of torch_binding.certify_inputs."""
    check_dim(emissions, 3, "emissions")
    check_dim(predictions, 3, "predictions")
    check_dim(frames, 2, "frames")
    check_dim(positions, 2, "positions")
    if emissions.dtype is torch.bfloat16:
        check_type(predictions, torch.bfloat16, "predictions")
    else:
        check_type(emissions, torch.float32, "emissions")
        check_type(predictions, torch.float32, "predictions")
    check_type(frames, torch.int32, "frames")
    check_type(positions, torch.int32, "positions")
    check_contiguous(frames, "frames")
    check_contiguous(positions, "positions")
    batch = emissions.shape[0]
    if emissions.shape[2] != predictions.shape[2]:
        raise ValueError("vocab size mismatch.")
    if predictions.shape[0] != batch:
        raise ValueError("must have predictions per example.")
    if frames.shape[0] != batch:
        raise ValueError("must have nodes per example.")
    if frames.shape != positions.shape:
        raise ValueError("frames and positions must have the same shape.")
    check_device(emissions, predictions, frames, positions)


def certify_indices(emissions, predictions, frames, positions, words=None):
    """That no frame, position or listed word lies beyond its tensor: after the kernels are enqueued one
    small kernel and one synchronisation tell the greatest.  (The kernels themselves take such an
    index for none, so a call with too great ones may run before it is refused.)  Inside `OnDevice`."""
    if frames.numel() == 0:
        return
    scratch = torch.empty(_transducer.node_summary_scratch_bytes, dtype=torch.uint8,
                          device=emissions.device)
    frame, position, word = _transducer.node_summary(
        frames.data_ptr(), positions.data_ptr(), frames.numel(),
        0 if words is None else words.data_ptr(), 0 if words is None else words.numel(),
        scratch.data_ptr())
    if frame >= emissions.shape[1]:
        raise ValueError("Frame index mismatch")
    if position >= predictions.shape[1]:
        raise ValueError("Position index mismatch")
    if word >= emissions.shape[2]:
        raise ValueError("Word index mismatch")


class OnDevice(object):
    """torch_binding.DeviceManager for calls that take a few microseconds: the device is switched only
    where it is another one."""

    def __init__(self, device):
        if device.type != "cuda":
            raise ValueError("transducer_b200 runs on CUDA tensors only (got %s)" % device)
        self.index = device.index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        _transducer.set_stream(torch._C._cuda_getCurrentRawStream(self.index))

    def __exit__(self, exc_type, exc_value, traceback):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def check_device(first, *others):
    device = first.device
    for t in others:
        if t.device != device:
            raise ValueError("all inputs must be on the same device.")


def check_no_tangents(*scores):
    """For results that are not differentiable: a tangent (forward-mode differentiation) would be lost."""
    if forward_ad._current_level < 0:
        return
    for x in scores:
        if forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError("this call has no derivatives and takes no tangents")


def check_temperature(temperature):
    if not 1e-38 <= temperature <= 1e30:
        raise ValueError("temperature must be positive, at least 1e-38 and at most 1e30")


def _rows(scores):
    """`scores` with the words of a row next to each other: itself wherever it is so laid out."""
    return scores if scores.stride(2) == 1 or scores.shape[2] == 1 else scores.contiguous()


def _describe(emissions, predictions, frames):
    """What the native calls want to know of the scores, and the sizes B, T, U, V, N."""
    B, T, V = emissions.shape
    e, p = emissions.stride(), predictions.stride()
    return ((emissions.data_ptr(), predictions.data_ptr(), emissions.dtype is torch.bfloat16,
             e[0], e[1], p[0], p[1]), (B, T, predictions.shape[1], V, frames.shape[1]))


def top_words(emissions, predictions, frames, positions, k, temperature=1.0, validate_nodes=True):
    """The ``k`` best words of every node (at most 256): what a beam search extends, and what a
    teacher records for `NodeDistillationLoss`.

    Returns words int32 [B, N, k] (the greater score first, of equal ones the lower word), their
    logits float32 [B, N, k] = scores / temperature, and rest float32 [B, N], the log-sum-exp of
    scores / temperature over all other words (-inf where there are none).  Where there is no node:
    -1, -inf, -inf.  They are detached from the inputs' graph: nothing here is differentiable (the
    log-probability of a word with gradients is minus the cost of `NodeDistillationLoss` with that
    word listed alone).  ``validate_nodes=False`` skips the check of the indices, which waits for the
    kernels, so that the call only enqueues work."""
    certify_nodes(emissions, predictions, frames, positions)
    check_no_tangents(emissions, predictions)
    check_temperature(temperature)
    if not 1 <= k <= min(MAX_LISTED_WORDS, emissions.shape[2]):
        raise ValueError("k must be between 1 and min(%d, vocabulary)" % MAX_LISTED_WORDS)
    emissions, predictions = _rows(emissions), _rows(predictions)
    B, N = frames.shape
    device = emissions.device
    with OnDevice(device):
        words = torch.empty((B, N, k), device=device, dtype=torch.int32)
        logits = torch.empty((B, N, k), device=device, dtype=torch.float32)
        rest = torch.empty((B, N), device=device, dtype=torch.float32)
        scores, sizes = _describe(emissions, predictions, frames)
        _transducer.top_words(scores, frames.data_ptr(), positions.data_ptr(), words.data_ptr(),
                              logits.data_ptr(), rest.data_ptr(), sizes, k, temperature)
        if validate_nodes:
            certify_indices(emissions, predictions, frames, positions)
    return words, logits, rest


def sample_words(emissions, predictions, frames, positions, uniforms, temperature=1.0, top_k=0,
                 top_p=1.0, min_p=0.0, validate_nodes=True):
    """A word of every node, drawn with the numbers ``uniforms`` float32 [B, N] in [0, 1).

    The scores are divided by ``temperature`` (0: the best word is taken); only the ``top_k`` best
    words stay (0: all), of them the fewest that have at least ``top_p`` of their probability, of
    them those with at least ``min_p`` of the best word's.  The word is the first, in the order of
    the vocabulary, up to which the probabilities that stay add up to more than the number's share
    of their sum; the comparisons come out as in 64-bit arithmetic.

    Returns words int32 [B, N] and log_probs float32 [B, N], the logarithm of the word's
    probability among those that stay.  Where there is no node: -1 and 0; where every word is
    masked: -1 and -inf; where a score is NaN or +inf: -1 and NaN.  Draws on the same inputs give
    the same words.  Both results are detached; ``validate_nodes``: see `top_words`."""
    certify_nodes(emissions, predictions, frames, positions)
    check_no_tangents(emissions, predictions)
    check_dim(uniforms, 2, "uniforms")
    check_type(uniforms, torch.float32, "uniforms")
    check_contiguous(uniforms, "uniforms")
    if uniforms.shape != frames.shape:
        raise ValueError("must have a number per node.")
    check_device(emissions, uniforms)
    if temperature != 0.0:
        check_temperature(temperature)
    if top_k < 0:
        raise ValueError("top_k must not be negative")
    if not 0.0 < top_p <= 1.0:
        raise ValueError("top_p must be above 0 and at most 1")
    if not 0.0 <= min_p <= 1.0:
        raise ValueError("min_p must be between 0 and 1")
    emissions, predictions = _rows(emissions), _rows(predictions)
    device = emissions.device
    with OnDevice(device):
        words = torch.empty(frames.shape, device=device, dtype=torch.int32)
        log_probs = torch.empty(frames.shape, device=device, dtype=torch.float32)
        scores, sizes = _describe(emissions, predictions, frames)
        _transducer.sample_words(scores, frames.data_ptr(), positions.data_ptr(),
                                 uniforms.data_ptr(), words.data_ptr(), log_probs.data_ptr(), sizes,
                                 temperature, min(top_k, sizes[3]), top_p, min_p)
        if validate_nodes:
            certify_indices(emissions, predictions, frames, positions)
    return words, log_probs


class NodeDistillation(torch.autograd.Function):
    """Autograd node for the distillation costs."""

    @staticmethod
    def forward(ctx, emissions, predictions, frames, positions, words, logits, rest, temperature,
                save, validate_nodes):
        emissions, predictions = _rows(emissions), _rows(predictions)
        device = emissions.device
        K = words.shape[2]
        with OnDevice(device):
            costs = torch.empty(frames.shape, device=device, dtype=torch.float32)
            scores, sizes = _describe(emissions, predictions, frames)
            nbytes = _transducer.distill_saved_bytes(*sizes[:3], sizes[4], K) if save else 0
            saved = _workspace(nbytes, device) if save else None
            _transducer.distill_forward(
                scores, frames.data_ptr(), positions.data_ptr(), words.data_ptr(),
                logits.data_ptr(), 0 if rest is None else rest.data_ptr(), costs.data_ptr(),
                saved.data_ptr() if save else 0, nbytes, sizes, K, temperature)
            if validate_nodes:
                certify_indices(emissions, predictions, frames, positions, words)
        if save:
            ctx.save_for_backward(emissions, predictions, frames, positions, words, saved)
            ctx.temperature = temperature
        return costs

    @staticmethod
    def backward(ctx, deltas):
        emissions, predictions, frames, positions, words, saved = ctx.saved_tensors
        device = emissions.device
        deltas = deltas.contiguous()
        need_e, need_p = ctx.needs_input_grad[:2]
        with OnDevice(device):
            egrads = torch.empty(emissions.shape, device=device, dtype=emissions.dtype) if need_e else None
            pgrads = torch.empty(predictions.shape, device=device, dtype=predictions.dtype) if need_p else None
            scores, sizes = _describe(emissions, predictions, frames)
            nbytes = _transducer.distill_backward_workspace_bytes(*sizes)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
            _transducer.distill_backward(
                scores, frames.data_ptr(), positions.data_ptr(), words.data_ptr(),
                saved.data_ptr(), saved.numel(), deltas.data_ptr(),
                0 if egrads is None else egrads.data_ptr(),
                0 if pgrads is None else pgrads.data_ptr(), sizes, words.shape[2],
                ctx.temperature, ws.data_ptr(), nbytes)
        if torch.is_grad_enabled():   # (somebody wants to differentiate these)
            egrads, pgrads = Once.apply(egrads, pgrads, emissions, predictions, deltas)
        return (egrads, pgrads) + (None,) * 8


class Once(torch.autograd.Function):
    """Gradients that are not differentiable again: asking for it is an error, not 0."""

    @staticmethod
    def forward(ctx, egrads, pgrads, *what_they_depend_on):
        return tuple(None if g is None else g.view_as(g) for g in (egrads, pgrads))

    @staticmethod
    def backward(ctx, *deltas):
        raise RuntimeError("the distillation cost is differentiable once only")


class NodeDistillationLoss(torch.nn.Module):
    """Distillation of a student joiner from a teacher's recorded best words, node by node: the
    Kullback-Leibler divergence from the teacher's distribution over the words it lists, and over
    "any other word" as one more outcome where the record says how much those weigh, to the
    student's softmax of (emissions + predictions) / temperature.

    With one listed word per node the cost is minus the student's log-probability of it.

    Arguments:
        temperature (float, optional): divides the student's scores.  The teacher's logits are taken
            as they are: `top_words` with the same temperature has divided them already.
        validate_nodes (bool, optional): check that no index lies beyond its tensor (default; waits
            for the forward kernels and reads three numbers back).  Pass False for a call that only
            enqueues work and can be captured in a CUDA graph (with its backward pass by
            torch.autograd.grad: `Tensor.backward` adds to a leaf on the stream on which the leaf
            was first used, which the capture does not see).
        reduction (str, optional): "none" (default), "sum" or "mean", the latter over the nodes
            that there are.
    """

    def __init__(self, temperature=1.0, validate_nodes=True, reduction="none"):
        super(NodeDistillationLoss, self).__init__()
        if reduction not in ("none", "sum", "mean"):
            raise ValueError("reduction must be 'none', 'sum' or 'mean'")
        check_temperature(temperature)
        self.temperature = temperature
        self.validate_nodes = validate_nodes
        self.reduction = reduction

    def forward(self, emissions, predictions, frames, positions, words, logits, rest=None):
        """
        emissions, predictions, frames, positions  the student's nodes (see the module's docstring)
        words   int32 [B, N, K]    the teacher's listed words, K <= 256; a negative one is ignored,
                                   equal ones of a node add up
        logits  float32 [B, N, K]  the teacher's logits for them (gradients w.r.t. them and rest: refused)
        rest    float32 [B, N], optional  log-sum-exp of the teacher's logits over all other words
                                   (without it the teacher's distribution is the listed words' alone)
        Returns costs float32 [B, N] (0 where there is no node or nothing is listed, +inf where the
        student masks a word that the teacher does not), differentiable once w.r.t. emissions and
        predictions.  The gradients are added up in the nodes' order and are the same bits from run
        to run.
        """
        certify_nodes(emissions, predictions, frames, positions)
        check_dim(words, 3, "words")
        check_dim(logits, 3, "logits")
        check_type(words, torch.int32, "words")
        check_type(logits, torch.float32, "logits")
        check_contiguous(words, "words")
        check_contiguous(logits, "logits")
        if words.shape != logits.shape:
            raise ValueError("words and logits must have the same shape.")
        if words.shape[:2] != frames.shape:
            raise ValueError("must have listed words per node.")
        if not 1 <= words.shape[2] <= MAX_LISTED_WORDS:
            raise ValueError("must list between 1 and %d words." % MAX_LISTED_WORDS)
        check_device(emissions, words, logits)
        if rest is not None:
            check_dim(rest, 2, "rest")
            check_type(rest, torch.float32, "rest")
            check_contiguous(rest, "rest")
            if rest.shape != frames.shape:
                raise ValueError("must have a rest per node.")
            check_device(emissions, rest)
        save = torch.is_grad_enabled()
        if save:
            if logits.requires_grad or (rest is not None and rest.requires_grad):
                raise ValueError("the costs are not differentiable w.r.t. the teacher's record: detach logits and rest")
            save = emissions.requires_grad or predictions.requires_grad
        costs = NodeDistillation.apply(emissions, predictions, frames, positions, words, logits,
                                       rest, self.temperature, save, self.validate_nodes)
        if self.reduction == "sum":
            return costs.sum()
        if self.reduction == "mean":
            here = ((frames >= 0) & (frames < emissions.shape[1])
                    & (positions >= 0) & (positions < predictions.shape[1]))
            return costs.sum() / here.sum().clamp(min=1)
        return costs
