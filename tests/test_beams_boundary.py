"""CPU tests of extend_beams, reorder_states and embed_words: what they refuse, in Python and in the C ABI, and the
generator's published answers.  No kernel is launched."""
import ctypes

import numpy as np
import pytest
import torch

import beam_reference as ref
from test_nodes_boundary import BAD_NODES, nodes
from transducer_b200 import _lib, embed_words, extend_beams, reorder_states
from transducer_b200.beams import _check_apart, _row

lib = _lib.lib
P = ctypes.c_void_p(64)   # (never followed: no kernel is launched)


@pytest.mark.parametrize("at,bad,kind,message", BAD_NODES)
def test_bad_nodes(at, bad, kind, message):
    a = nodes()
    a[at] = bad
    with pytest.raises(kind, match=message):
        extend_beams(*a, torch.zeros(2, 4), 2)


@pytest.mark.parametrize("bad,kind,message", [
    (torch.zeros(2, 4, 1), ValueError, "scores must be 2D"),
    (torch.zeros(2, 4, dtype=torch.float64), TypeError, "scores must be torch.float32"),
    (torch.zeros(2, 3), ValueError, "a score per node"),
    (torch.zeros(4, 2).t(), ValueError, "scores must be contiguous"),
    (torch.zeros(2, 4, device="meta"), ValueError, "same device")])
def test_bad_scores(bad, kind, message):
    with pytest.raises(kind, match=message):
        extend_beams(*nodes(), bad, 2)


@pytest.mark.parametrize("width", [0, -1, 257])
def test_bad_width(width):
    with pytest.raises(ValueError, match="width must be between"):
        extend_beams(*nodes(), torch.zeros(2, 4), width)


def test_cpu_tensors_are_refused():
    parents = torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: extend_beams(*nodes(), torch.zeros(2, 4), 2),
                 lambda: reorder_states(torch.zeros(2, 4, 5), parents),
                 lambda: embed_words(torch.zeros(3, 4), parents)):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()


def test_tangents_are_refused():
    import torch.autograd.forward_ad as forward
    with forward.dual_level():
        for at in range(2):
            a = nodes()
            a[at] = forward.make_dual(a[at], torch.ones_like(a[at]))
            with pytest.raises(RuntimeError, match="no tangents"):
                extend_beams(*a, torch.zeros(2, 4), 2)
        dual = forward.make_dual(torch.zeros(2, 4), torch.ones(2, 4))
        with pytest.raises(RuntimeError, match="no tangents"):
            extend_beams(*nodes(), dual, 2)
        with pytest.raises(RuntimeError, match="no tangents"):
            reorder_states(dual, torch.zeros(2, 3, dtype=torch.int32))
        with pytest.raises(RuntimeError, match="no tangents"):
            embed_words(dual, torch.zeros(2, 3, dtype=torch.int32))


def test_bad_parents_and_states():
    parents = torch.zeros(2, 3, dtype=torch.int32)
    s = torch.zeros(2, 4, 5)
    cases = [
        (s, parents.long(), None, TypeError, "parents must be torch.int32"),
        (s, parents[0], None, ValueError, "parents must be 2D"),
        (s, torch.zeros(3, 2, dtype=torch.int32).t(), None, ValueError, "parents must be contiguous"),
        ([], parents, None, ValueError, "must be a state"),
        ([s[0, 0]], parents, None, ValueError, "dimension of utterances"),
        ([s, s[:1]], parents, None, ValueError, "states per example"),
        ([s, s[:, :3]], parents, None, ValueError, "same number of hypotheses"),
        ([s, s.to("meta")], parents, None, ValueError, "same device"),
        ([s], parents, [s[:, :3], s], ValueError, "an output per state"),
        (s, parents, s[:, :3].double(), TypeError, "the states' types"),
        (s, parents, s, ValueError, "shape of the reordered"),
        (s, parents, torch.zeros(2, 3, 10)[..., ::2], ValueError, "contiguous behind"),
        (s, parents, torch.zeros(2, 3, 5, requires_grad=True), ValueError, "not require gradients"),
        (s, parents, torch.zeros(2, 3, 5, device="meta"), ValueError, "same device"),
    ]
    for states, p, out, kind, message in cases:
        with pytest.raises(kind, match=message):
            reorder_states(states, p, out=out)


def test_outputs_that_overlap():
    parents = torch.zeros(2, 4, dtype=torch.int32)

    def accept(states, out, W):
        _check_apart([_row(s) for s in states], out, states[0].shape[0], states[0].shape[1], W, parents)

    def refuse(states, out, message):
        with pytest.raises(ValueError, match=message):
            accept(states, out, out[0].shape[1])
    room = torch.zeros(2, 9, 5)
    s = room[:, :4]
    accept([s], [s], 4)                       # in place
    accept([s], [room[:, :7]], 7)             # in place, more of them
    accept([s], [s[:, :3]], 3)
    accept([s[:1]], [room[:1, 4:9]], 5)       # side by side
    accept([s], [torch.zeros(2, 3, 5)], 3)
    refuse([s], [room[:, 1:5]], "a state itself or not overlap")
    refuse([s], [room[:, 4:8]], "a state itself or not overlap")   # (between the utterances' rows)
    refuse([s, torch.zeros(2, 4, 5)], [torch.zeros(2, 4, 5), s], "a state itself or not overlap")
    refuse([room[:, :3], room[:, 3:6]], [room[:, :6], torch.zeros(2, 6, 5)], "a state itself or not overlap")
    o = torch.zeros(2, 4, 5)
    refuse([s, s], [o, o], "with each other")
    refuse([s], [torch.zeros(2, 1, 5).expand(2, 4, 5)], "with itself")
    refuse([s], [torch.zeros(1, 4, 5).expand(2, 4, 5)], "with itself")
    refuse([s], [torch.zeros(32).as_strided((2, 4, 5), (15, 4, 1))], "with itself")
    refuse([parents], [parents], "with parents")
    big = torch.zeros(1, 4097, 1)
    refuse([big], [big], "at most 4096")


def test_numbers_together():
    x = torch.zeros(2, 3, 4, 5)
    assert _row(x)[1:] == (240, 80, 80) and _row(x[:, ::2])[1:] == (240, 160, 80)
    assert _row(x.transpose(0, 1))[1:] == (80, 240, 80) and _row(x[..., :1, :])[1:] == (240, 80, 20)
    assert _row(x[..., 0, 0])[1:] == (240, 80, 4) and _row(x[:, :, :0])[3] == 0
    assert _row(x[..., ::2]) is None and _row(x.transpose(2, 3)) is None and _row(x[:, :, ::2]) is None


@pytest.mark.parametrize("change,kind,message", [
    (dict(table=torch.zeros(3)), ValueError, "table must be 2D"),
    (dict(table=torch.zeros(3, 4, dtype=torch.float16)), TypeError, "table must be torch.float32"),
    (dict(words=torch.zeros(2, 3)), TypeError, "words must be torch.int32"),
    (dict(words=torch.zeros(2, 3, dtype=torch.int64)), TypeError, "words must be torch.int32"),
    (dict(words=torch.zeros(3, 2, dtype=torch.int32).t()), ValueError, "words must be contiguous"),
    (dict(words=torch.zeros(2, 3, dtype=torch.int32, device="meta")), ValueError, "same device"),
    (dict(scale=float("inf")), ValueError, "scale must be finite"),
    (dict(scale=float("nan")), ValueError, "scale must be finite"),
    (dict(dropout=1.0, seed=1), ValueError, "dropout must be"),
    (dict(dropout=-0.1, seed=1), ValueError, "dropout must be"),
    (dict(dropout=float("nan"), seed=1), ValueError, "dropout must be"),
    (dict(dropout=0.1), ValueError, "needs a seed"),
    (dict(dropout=0.1, seed=2 ** 63), ValueError, "64 bits"),
    (dict(dropout=0.1, seed=torch.zeros(1)), TypeError, "seed must be torch.int64"),
    (dict(dropout=0.1, seed=torch.zeros(2, dtype=torch.int64)), ValueError, "one number"),
    (dict(dropout=0.1, seed=torch.zeros(1, dtype=torch.int64, device="meta")), ValueError, "same device"),
])
def test_bad_embeddings(change, kind, message):
    args = dict(table=torch.zeros(3, 4), words=torch.zeros(2, 3, dtype=torch.int32))
    args.update(change)
    with pytest.raises(kind, match=message):
        embed_words(**args)


def refused(rc, message):
    assert rc == 1
    assert message in lib.tb200_last_error().decode()


def extend_abi(B=1, T=2, U=2, V=8, N=2, width=2, strides=(16, 8, 16, 8), ws=P, nbytes=1 << 20):
    return lib.tb200_extend_beams(P, P, 0, *strides, P, P, P, P, P, P, B, T, U, V, N, width, None, ws, nbytes)


@pytest.mark.parametrize("change,message", [
    (dict(B=-1), "negative"), (dict(V=0), "negative"), (dict(N=-1), "negative"),
    (dict(strides=(16, -8, 16, 8)), "negative stride"), (dict(width=0), "between 1 and 256"),
    (dict(width=257), "between 1 and 256"), (dict(V=(1 << 28) + 1), "alphabet"),
    (dict(B=1 << 16, N=1 << 15), "too many nodes"), (dict(nbytes=16), "workspace too small"),
    (dict(ws=None), "workspace too small"), (dict(ws=ctypes.c_void_p(72)), "aligned")])
def test_abi_refuses_to_extend(change, message):
    refused(extend_abi(**change), message)


class Moved(ctypes.Structure):
    _fields_ = [("from_", ctypes.c_void_p), ("to", ctypes.c_void_p)] + [
        (n, ctypes.c_longlong) for n in ("fromStrideB", "fromStrideN", "toStrideB", "toStrideN", "rowBytes")]


@pytest.mark.parametrize("state,sizes,message", [
    ((64, 128, 8, 8, 8, 8, -1), (1, 2, 2), "negative"), ((64, 128, 8, -8, 8, 8, 8), (1, 2, 2), "negative"),
    ((64, 128, 8, 8, 8, 8, 8), (-1, 2, 2), "negative"), ((64, 128, 8, 8, 8, 8, 8), (1, 2, -1), "negative"),
    ((64, 64, 16, 8, 24, 8, 8), (2, 2, 3), "keep their strides"),
    ((64, 64, 16, 8, 16, 8, 8), (1, 2, 4097), "4096"),
    ((64, 128, 16, 8, 16, 8, 8), (1 << 16, 1 << 15, 2), "too many hypotheses"),
    ((64, 128, 16, 8, 16, 8, 1 << 50), (1, 2, 2), "too large")])
def test_abi_refuses_to_reorder(state, sizes, message):
    refused(lib.tb200_reorder_states(ctypes.byref(Moved(*state)), 1, P, *sizes, 0, None), message)


@pytest.mark.parametrize("change,message", [
    (dict(count=-1), "negative"), (dict(R=-1), "negative"), (dict(H=-1), "negative"), (dict(stride=-4), "negative"),
    (dict(count=1 << 31), "too many words"), (dict(R=(1 << 28) + 1), "2^28 rows"), (dict(H=(1 << 23) + 1), "2^23"),
    (dict(dropout=1.0), "dropout"), (dict(dropout=float("nan")), "dropout"), (dict(scale=float("inf")), "scale"),
    (dict(scale=1e39), "scale")])
def test_abi_refuses_to_embed(change, message):
    a = dict(stride=4, count=2, R=3, H=4, scale=1.0, dropout=0.0)
    a.update(change)
    refused(lib.tb200_embed_words(P, 0, a["stride"], P, a["count"], P, a["R"], a["H"], a["scale"], a["dropout"], 0,
                                  None, None), message)
    if "stride" not in change:
        refused(lib.tb200_embed_backward(P, 0, P, a["count"], P, a["R"], a["H"], a["scale"], a["dropout"], 0, None,
                                         P, 1 << 40), message)


def test_abi_wants_workspace_for_gradients():
    n = lib.tb200_embed_backward_workspace_bytes(1000, 30, 8)
    refused(lib.tb200_embed_backward(P, 0, P, 1000, P, 30, 8, 1.0, 0.0, 0, None, P, n - 1), "workspace too small")


def test_published_answers_of_the_generator():
    """The known answers that the generator's authors publish with it (Random123, philox4x32 with 10 rounds)."""
    ones = 0xffffffff
    cases = [((0,) * 4, (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
             ((ones,) * 4, (ones, ones), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
             ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
              (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]
    for counter, key, want in cases:
        got = ref.philox(np.array(counter, np.uint64), key)
        assert tuple(int(x) for x in got) == want


@pytest.mark.parametrize("dropout", [0.1, 0.5, 0.9, 1e-6])
def test_share_that_stays(dropout):
    """Within five standard deviations, and the numbers of a group and of neighbours are not alike."""
    H, count = 96, 2000
    k = round(dropout * 65536) / 65536
    stays = ref.kept(count, H, dropout, 12345).double()
    n = stays.numel()
    assert abs(stays.sum().item() - n * (1 - k)) <= 5 * (n * k * (1 - k)) ** 0.5
    if k > 0.05:
        for shift in (1, 2, 4, 8):
            a, b = stays[:, shift:].flatten() - (1 - k), stays[:, :-shift].flatten() - (1 - k)
            assert abs((a * b).mean().item()) <= 5 * k * (1 - k) / a.numel() ** 0.5
