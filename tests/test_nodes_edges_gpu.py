"""Node operators (transducer_b200.nodes) at the edges of what their documentation allows."""

import pytest
import torch

from test_nodes_gpu import UNIT, check_sample, make
from transducer_b200 import sample_words

pytestmark = pytest.mark.gpu


# ---- draws among words of next to no weight ---------------------------------------------------

def test_draw_of_the_first_word_however_small():
    """A number of 0 takes the first word that has any weight in 64 bits, 2^-130 of the best one's here."""
    E = torch.tensor([[[-9.0, 0.0, -0.1]]]).cuda()
    zero = torch.zeros(1, 1, dtype=torch.int32).cuda()
    word, log_prob = sample_words(E, torch.zeros_like(E), zero, zero, torch.zeros(1, 1).cuda(), temperature=0.1)
    assert word.item() == 0
    z = torch.tensor([-9.0, 0.0, torch.tensor(-0.1).item()], dtype=torch.float64) / 0.1
    assert abs(log_prob.item() - torch.log_softmax(z, 0)[0].item()) <= 100 * 2 * UNIT


SMALL_RULES = [dict(), dict(top_k=2), dict(top_k=17), dict(top_k=400), dict(min_p=1e-30), dict(min_p=1e-40),
               dict(min_p=1e-200), dict(top_k=40, min_p=1e-60), dict(top_p=0.99), dict(top_k=30, top_p=0.9)]


@pytest.mark.parametrize("V", [3, 100, 520, 1025, 5000, 20000, 60000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_draws_with_the_smallest_numbers(V, dtype):
    """Temperatures at which most words have weights below 2^-126, and numbers down to 0."""
    N = 12
    E, P, frames, positions, g = make(2, 6, 4, V, N, dtype, seed=V + 2, holes=False)
    numbers = torch.tensor([0.0, 1e-45, 1e-42, 1e-38, 1e-35, 1e-30, 1e-20, 1e-8, 0.5, 1.0 - 2.0 ** -24, 0.0, 0.0])
    uniforms = numbers[torch.stack([torch.randperm(N, generator=g) for _ in range(2)])].cuda()
    for temperature in (0.3, 0.1, 0.04):
        for rule in SMALL_RULES:
            check_sample(E, P, frames, positions, uniforms, temperature=temperature, **rule)
