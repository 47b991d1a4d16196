"""examples/policy_experts.py runs all four row operators with the Muon step, and learns."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "policy_experts.py")


def test_policy_example_earns_reward():
    spec = importlib.util.spec_from_file_location("policy_experts", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    rewards = example.train(steps=24, log=lambda line: None)
    # chance is one in 64; 64 answers of 10 tokens a step: three times that is far outside chance
    assert rewards[0] < 3 / example.VOCAB
    assert sum(rewards[-4:]) / 4 > 6 / example.VOCAB
