"""CPU tests of the node operators' boundary: what they refuse, in Python and in the C ABI.  No kernel
is launched."""
import ctypes

import pytest
import torch

from transducer_b200 import NodeDistillationLoss, _lib, sample_words, top_words

lib = _lib.lib


def nodes(B=2, T=5, U=3, V=8, N=4, dtype=torch.float32):
    return [torch.zeros(B, T, V, dtype=dtype), torch.zeros(B, U, V, dtype=dtype),
            torch.zeros(B, N, dtype=torch.int32), torch.zeros(B, N, dtype=torch.int32)]


def record(B=2, N=4, K=3):
    return [torch.zeros(B, N, K, dtype=torch.int32), torch.zeros(B, N, K)]


BAD_NODES = [
    (0, torch.zeros(5, 8), ValueError, "emissions must be 3D"),
    (1, torch.zeros(2, 3), ValueError, "predictions must be 3D"),
    (2, torch.zeros(4, dtype=torch.int32), ValueError, "frames must be 2D"),
    (3, torch.zeros(2, 4, 1, dtype=torch.int32), ValueError, "positions must be 2D"),
    (0, torch.zeros(2, 5, 8, dtype=torch.float16), TypeError, "emissions must be torch.float32"),
    (1, torch.zeros(2, 3, 8, dtype=torch.bfloat16), TypeError, "predictions must be torch.float32"),
    (0, torch.zeros(2, 5, 8, dtype=torch.bfloat16), TypeError, "predictions must be torch.bfloat16"),
    (2, torch.zeros(2, 4, dtype=torch.int64), TypeError, "frames must be torch.int32"),
    (3, torch.zeros(2, 4), TypeError, "positions must be torch.int32"),
    (2, torch.zeros(4, 2, dtype=torch.int32).t(), ValueError, "frames must be contiguous"),
    (1, torch.zeros(2, 3, 9), ValueError, "vocab size mismatch."),
    (1, torch.zeros(1, 3, 8), ValueError, "must have predictions per example."),
    (2, torch.zeros(3, 4, dtype=torch.int32), ValueError, "must have nodes per example."),
    (3, torch.zeros(2, 5, dtype=torch.int32), ValueError, "the same shape"),
    (3, torch.zeros(2, 4, dtype=torch.int32, device="meta"), ValueError, "same device"),
]


@pytest.mark.parametrize("at,bad,kind,message", BAD_NODES)
def test_bad_nodes(at, bad, kind, message):
    a = nodes()
    a[at] = bad
    for call in (lambda: top_words(*a, 2), lambda: sample_words(*a, torch.zeros(2, 4)),
                 lambda: NodeDistillationLoss()(*a, *record())):
        with pytest.raises(kind, match=message):
            call()


def test_cpu_tensors_are_refused():
    for call in (lambda: top_words(*nodes(), 2), lambda: sample_words(*nodes(), torch.zeros(2, 4)),
                 lambda: NodeDistillationLoss()(*nodes(), *record())):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            call()


@pytest.mark.parametrize("k", [0, -1, 9, 257])
def test_bad_k(k):
    with pytest.raises(ValueError, match="k must be between"):
        top_words(*nodes(), k)


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan"), float("inf"), 1e-40, 1e31])
def test_bad_temperature(temperature):
    with pytest.raises(ValueError, match="temperature must be positive"):
        top_words(*nodes(), 2, temperature=temperature)
    with pytest.raises(ValueError, match="temperature must be positive"):
        NodeDistillationLoss(temperature=temperature)
    if temperature != 0.0:
        with pytest.raises(ValueError, match="temperature must be positive"):
            sample_words(*nodes(), torch.zeros(2, 4), temperature=temperature)


@pytest.mark.parametrize("bad,kind,message", [
    (torch.zeros(2, 4, 1), ValueError, "uniforms must be 2D"),
    (torch.zeros(2, 4, dtype=torch.float64), TypeError, "uniforms must be torch.float32"),
    (torch.zeros(2, 3), ValueError, "a number per node"),
    (torch.zeros(4, 2).t(), ValueError, "uniforms must be contiguous"),
    (torch.zeros(2, 4, device="meta"), ValueError, "same device")])
def test_bad_uniforms(bad, kind, message):
    with pytest.raises(kind, match=message):
        sample_words(*nodes(), bad)


@pytest.mark.parametrize("rule,message", [
    (dict(top_k=-1), "top_k"), (dict(top_p=0.0), "top_p"), (dict(top_p=1.5), "top_p"),
    (dict(top_p=float("nan")), "top_p"), (dict(min_p=-0.1), "min_p"), (dict(min_p=1.1), "min_p"),
    (dict(min_p=float("nan")), "min_p")])
def test_bad_rules(rule, message):
    with pytest.raises(ValueError, match=message):
        sample_words(*nodes(), torch.zeros(2, 4), **rule)


def test_bad_records():
    words, logits = record()
    rest = torch.zeros(2, 4)
    cases = [
        (words.long(), logits, None, TypeError, "words must be torch.int32"),
        (words, logits.double(), None, TypeError, "logits must be torch.float32"),
        (words[0], logits, None, ValueError, "words must be 3D"),
        (words, logits[..., 0], None, ValueError, "logits must be 3D"),
        (words, logits[..., :2].contiguous(), None, ValueError, "the same shape"),
        (words[:, :3].contiguous(), logits[:, :3].contiguous(), None, ValueError, "listed words per node"),
        (words[..., :0], logits[..., :0], None, ValueError, "between 1 and 256 words"),
        (torch.zeros(2, 4, 257, dtype=torch.int32), torch.zeros(2, 4, 257), None, ValueError, "between 1 and 256"),
        (words.transpose(0, 1).contiguous().transpose(0, 1), logits, None, ValueError, "words must be contiguous"),
        (words, logits, rest.double(), TypeError, "rest must be torch.float32"),
        (words, logits, rest[:, :3].contiguous(), ValueError, "a rest per node"),
        (words, logits, rest[0], ValueError, "rest must be 2D"),
        (words, logits, rest.to("meta"), ValueError, "same device"),
    ]
    for w, l, r, kind, message in cases:
        with pytest.raises(kind, match=message):
            NodeDistillationLoss()(*nodes(), w, l, r)
    with pytest.raises(ValueError, match="reduction"):
        NodeDistillationLoss(reduction="average")


@pytest.mark.parametrize("student", [False, True])
@pytest.mark.parametrize("which", [0, 1])
def test_records_that_want_gradients(which, student):
    words, logits = record()
    rest = torch.zeros(2, 4)
    (logits, rest)[which].requires_grad_(True)
    a = nodes()
    a[0].requires_grad_(student)
    with pytest.raises(ValueError, match="not differentiable w.r.t. the teacher's record"):
        NodeDistillationLoss()(*a, words, logits, rest)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA tensors only"):
        NodeDistillationLoss()(*a, words, logits, rest)


@pytest.mark.parametrize("which", [0, 1])
def test_tangents(which):
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        a = nodes()
        for call in (lambda: top_words(*a, 2), lambda: sample_words(*a, torch.zeros(2, 4))):
            with pytest.raises(ValueError, match="CUDA tensors only"):
                call()
        a[which] = forward_ad.make_dual(a[which], torch.ones_like(a[which]))
        for call in (lambda: top_words(*a, 2), lambda: sample_words(*a, torch.zeros(2, 4))):
            with pytest.raises(RuntimeError, match="no tangents"):
                call()
        with pytest.raises((RuntimeError, ValueError)):
            NodeDistillationLoss()(*a, *record())


# ---- the C ABI: every refusal comes before the first CUDA call ------------------------------

def test_c_abi_refusals():
    strides = (40, 8, 24, 8)

    def top(B=2, T=5, U=3, V=8, N=4, k=2, temperature=1.0, strides=strides):
        return lib.tb200_top_words(None, None, 0, *strides, None, None, None, None, None, B, T, U, V, N, k,
                                   temperature)

    for bad in (dict(B=-1), dict(T=-1), dict(U=-1), dict(V=0), dict(N=-1), dict(k=0), dict(k=9), dict(k=257, V=400),
                dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=1e-60), dict(temperature=1e31),
                dict(B=1 << 16, N=1 << 15), dict(B=1 << 16, T=1 << 15, N=0), dict(B=1 << 16, U=1 << 15, N=0), dict(V=(1 << 28) + 1),
                dict(strides=(-40, 8, 24, 8))):
        assert top(**bad) == 1, bad
        assert lib.tb200_last_error()
    assert top(B=0) == 0 and top(N=0) == 0

    def sample(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, B=2):
        return lib.tb200_sample_words(None, None, 1, *strides, None, None, None, None, None, B, 5, 3, 8, 4,
                                      temperature, top_k, top_p, min_p)

    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.01), dict(min_p=-0.5),
                dict(min_p=2.0), dict(top_p=float("nan")), dict(min_p=float("nan"))):
        assert sample(**bad) == 1, bad
    assert sample(B=0, temperature=0.0) == 0

    saved = lib.tb200_distill_saved_bytes(2, 5, 3, 4, 3)
    assert saved >= 2 * 4 * (16 + 12) and lib.tb200_distill_saved_bytes(0, 5, 3, 4, 3) == 0
    some = ctypes.c_void_p(256)
    most = (ctypes.c_int * 3)()
    assert lib.tb200_node_summary(None, None, -1, None, 0, some, most) == 1
    assert lib.tb200_node_summary(None, None, 4, None, 0, None, most) == 1
    assert lib.tb200_node_summary_scratch_bytes() >= 12

    def forward(K=3, V=8, saved_bytes=saved, rest=None, B=2):
        return lib.tb200_distill_forward(None, None, 0, *strides, None, None, None, None, rest, None, some,
                                         saved_bytes, B, 5, 3, V, 4, K, 1.0)

    for bad in (dict(K=0), dict(K=257), dict(saved_bytes=saved - 1), dict(V=(1 << 28) + 1, rest=some)):
        assert forward(**bad) == 1, bad
    assert forward(B=0) == 0

    need = lib.tb200_distill_backward_workspace_bytes(2, 5, 3, 8, 4)
    assert need > 0

    def backward(saved=some, saved_bytes=saved, ws=some, ws_bytes=need, B=2):
        return lib.tb200_distill_backward(None, None, 0, *strides, None, None, None, saved, saved_bytes, None, None,
                                          None, B, 5, 3, 8, 4, 3, 1.0, ws, ws_bytes)

    odd = ctypes.c_void_p(264)
    for bad in (dict(saved=None), dict(saved_bytes=saved - 1), dict(saved=odd), dict(ws=odd), dict(ws=None), dict(ws_bytes=need - 1)):
        assert backward(**bad) == 1, bad
    assert backward(B=0, saved_bytes=0) == 0


def test_workspaces_do_not_grow_for_smaller_calls():
    for f, sizes in ((lib.tb200_distill_saved_bytes, [(B, 50, 9, 40, 8) for B in range(30)]),
                     (lib.tb200_distill_saved_bytes, [(3, 50, 9, N, 8) for N in range(300)]),
                     (lib.tb200_distill_saved_bytes, [(3, 50, 9, 40, K) for K in range(1, 257)]),
                     (lib.tb200_distill_saved_bytes, [(3, T, 9, 40, 8) for T in range(600)]),
                     *((lib.tb200_distill_backward_workspace_bytes, sizes) for sizes in (
                         [(B, 300, 40, 600, 340) for B in range(120)], [(3, T, 9, 700, 400) for T in range(900)],
                         [(3, 9, U, 1000, 90) for U in range(300)], [(2, 90, 9, V, 99) for V in range(1, 9000, 7)],
                         [(2, 30, 9, 600, N) for N in range(900)]))):
        got = [f(*s) for s in sizes]
        assert got == sorted(got)
