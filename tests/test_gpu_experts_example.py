"""The routed-experts operators together, as the example uses them."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_balanced_experts_learn_and_share_the_tokens():
    spec = importlib.util.spec_from_file_location("balanced_experts", os.path.join(ROOT, "examples", "balanced_experts.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, busiest = example.train(steps=40, tokens=1024)
    assert losses[-1] < 0.5 * losses[0]
    _, alone = example.train(steps=40, tokens=1024, balance=False)
    assert busiest < 2.0 < alone
