"""reorder_states, extend_beams and embed_words on a GPU: calls beside those of test_beams_gpu.py."""
import pytest
import torch

import test_beams_gpu as base
from transducer_b200 import reorder_states

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
