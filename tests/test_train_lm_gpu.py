"""The example's training step: layer, norms, head loss and optimiser together."""
import importlib.util
import os

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "train_lm.py")


@pytest.fixture(scope="module")
def lm():
    spec = importlib.util.spec_from_file_location("train_lm", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("bits", [8, 32])
def test_it_learns(lm, bits):
    """From about log(vocabulary) towards what a tenth of random tokens leave: 0.1 log(1000) + 0.33 = 1.0."""
    losses = lm.train(steps=80, state_bits=bits)
    assert np.isfinite(losses).all() and losses[0] > 5.0
    assert np.mean(losses[-5:]) < 0.6 * losses[0]


def test_gradient_of_the_whole_step_against_differences(lm):
    """The loss at embeddings moved along the gradient, against the gradient's square: BF16 activations and weights decide the
    tolerance (2^-8 of values that add up over three products), routing changes of a few tokens the rest."""
    tokens, targets = lm.batch(16, 64, 1000, 5)
    model = lm.Model(blocks=1)
    base = model.embed.clone()
    model.step(tokens, targets, lr=0.0)
    grad = model.d_embed.clone()
    size = grad.norm()
    s = 0.02 * base.norm() / size
    ends = []
    for sign in (1, -1):
        model.embed.copy_(base + sign * s * grad)
        model.head.copy_(model.embed)
        ends.append(float(model.step(tokens, targets, lr=0.0)))
    want = float(2 * s * size ** 2)
    assert abs(ends[0] - ends[1] - want) <= 0.15 * want
    torch.cuda.synchronize()
