"""Rows of a table for words (`embed_words`): a prediction network's inputs, or the predictions themselves where
they depend on the word before alone.  The reference starts from given predictions and has no counterpart.

CUDA tensors only, like `TransducerLoss`; the work is enqueued on torch's current stream."""
import math

import torch

from . import _transducer
from .nodes import OnDevice, check_device, check_no_tangents
from .torch_binding import check_contiguous, check_dim, check_type


class WordEmbedding(torch.autograd.Function):
    """Autograd node for the rows."""

    @staticmethod
    def forward(ctx, table, words, scale, dropout, seed, validate_words):
        rows, numbers, place = _rows_of(table, words, scale, dropout, seed, validate_words)
        if place:
            ctx.save_for_backward(words, seed)
        else:
            ctx.save_for_backward(words)
        count, (R, H) = words.numel(), table.shape
        ctx.rest = (count, R, H, table.dtype is torch.bfloat16, scale, dropout, numbers,
                    _transducer.embed_backward_workspace_bytes(count, R, H))
        return rows

    @staticmethod
    def backward(ctx, deltas):
        # (refuses words, and a seed on the device, that were written since; hooks may bring them back as other tensors)
        words, *seed = ctx.saved_tensors
        count, R, H, bf16, scale, dropout, numbers, nbytes = ctx.rest
        check_device(deltas, words, *seed)
        place = seed[0].data_ptr() if seed else 0
        if not words.is_contiguous():
            words = words.contiguous()
        if deltas.is_neg():
            deltas = deltas.resolve_neg()
        if not deltas.is_contiguous():
            deltas = deltas.contiguous()
        with OnDevice(deltas.device):
            grad = deltas.new_empty((R, H))
            ws = words.new_empty(nbytes // 4 + 1) if nbytes else None   # (few words need none)
            _transducer.embed_backward(deltas.data_ptr(), bf16, words.data_ptr(), count, grad.data_ptr(), R, H, scale,
                                       dropout, numbers, place, ws.data_ptr() if nbytes else 0, nbytes)
        if torch.is_grad_enabled():   # (somebody wants to differentiate it)
            grad = Once.apply(grad, deltas)
        return (grad,) + (None,) * 5


class Once(torch.autograd.Function):
    """A gradient that is not differentiable again: asking for it is an error, not 0."""

    @staticmethod
    def forward(ctx, grad, deltas):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *deltas):
        raise RuntimeError("embedded words are differentiable once only")


def _seed(seed):
    """The seed as a number, and the address of one on the device (0: none)."""
    if isinstance(seed, torch.Tensor):
        return 0, seed.data_ptr()
    return 0 if seed is None else seed, 0


def _rows_of(table, words, scale, dropout, seed, validate_words):
    """The rows, and the seed as `_seed` has it."""
    if table.is_neg():   # (as for scores, see nodes.py)
        table = table.resolve_neg()
    if table.stride(1) != 1 and table.shape[1] != 1:
        table = table.contiguous()
    R, H = table.shape
    numbers, place = _seed(seed)
    with OnDevice(table.device):
        rows = table.new_empty(words.shape + (H,))
        beyond = _transducer.embed_words(table.data_ptr(), table.dtype is torch.bfloat16, table.stride(0),
                                         words.data_ptr(), words.numel(), rows.data_ptr(), R, H, scale, dropout,
                                         numbers, place, validate_words)
    if beyond:
        raise ValueError("Word index mismatch")
    return rows, numbers, place


def embed_words(table, words, scale=1.0, dropout=0.0, seed=None, validate_words=True):
    """The rows of ``table`` (float32 or bfloat16 [R, H]) for ``words`` (int32, any shape), times ``scale``:
    a tensor [*words.shape, H] of the table's type.  A negative word has a row of zeros.

    With ``dropout`` above 0 that share of the numbers, to the nearest 65536th, is dropped and the others
    are divided by what is left of 1.  Which ones follows from ``seed`` and a number's place alone (Philox4x32-10; the C
    ABI's header says how), so that no mask is stored, and the same seed drops the same places: take
    another one for every call.  It is a whole number, or one int64 on the device, which is read when the kernels run: a
    captured call whose seed is written between its replays drops other numbers each time.

    Differentiable once w.r.t. the table: the gradient is dense, its sums are made in fp32 in an order that follows
    from the words alone and are the same bits from run to run.  ``validate_words=False`` skips the check that no word is R or
    more (such ones have rows of zeros), which waits for the kernels, so that the call only enqueues work and
    can be captured in a CUDA graph (its backward pass by torch.autograd.grad, when no earlier graph of the
    table, such as rows of a call before, lives any more: torch would make the capture wait for that one's stream).

    Previous words of transcripts, as a prediction network takes them (0: the start symbol)::

        n = torch.arange(U + 1, device=labels.device)
        words = torch.nn.functional.pad(labels, (1, 0))
        words = words.masked_fill(n > label_lengths[:, None], -1)
    """
    check_dim(table, 2, "table")
    if table.dtype is not torch.bfloat16:
        check_type(table, torch.float32, "table")
    check_type(words, torch.int32, "words")
    check_contiguous(words, "words")
    check_device(table, words)
    check_no_tangents(table)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not 0.0 <= dropout < 1.0:
        raise ValueError("dropout must be at least 0 and below 1")
    if dropout > 0.0 and seed is None:
        raise ValueError("dropout needs a seed")
    if isinstance(seed, torch.Tensor):
        check_type(seed, torch.int64, "seed")
        if seed.numel() != 1:
            raise ValueError("seed must be one number")
        check_device(table, seed)
    elif seed is not None and not -2 ** 63 <= seed < 2 ** 63:
        raise ValueError("seed must fit 64 bits")
    if not (table.requires_grad and torch.is_grad_enabled()):
        return _rows_of(table, words, scale, dropout, seed, validate_words)[0]
    return WordEmbedding.apply(table, words, scale, dropout, seed, validate_words)
