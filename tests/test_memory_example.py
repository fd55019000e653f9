"""examples/memory_critic.py: the sequence operators together, on rollouts of a Sim."""
import importlib.util
import os

import numpy as np
import pytest
import torch

EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "memory_critic.py")


def example():
    spec = importlib.util.spec_from_file_location("memory_critic", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.gpu
def test_the_memory_critic_learns_and_acts_as_it_was_trained():
    """The loss falls, and ticks one at a time give the values and states of the rollout at once.

    Values are sums of 128 products of numbers of about 1 with weights of up to 1 / sqrt(128), from rows whose
    relative error is that of fp32 sums over 64 ticks: below 1e-4 with a wide margin."""
    _, losses, differ = example().train(envs=64, horizon=40, rollouts=3, epochs=6, log=lambda *a, **k: print(*a, **k))
    losses = np.array(losses)
    assert np.isfinite(losses).all()
    assert losses[-1, 1] < losses[0, 0]
    assert differ < 1e-4
