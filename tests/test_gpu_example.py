"""The example runs the operators together: the loss falls, and greedy decoding
reports the chosen token as the best alternative."""

import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "train_and_score.py")


def test_train_and_score(cuda_device):
    spec = importlib.util.spec_from_file_location("train_and_score", PATH)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    r = ex.main(steps=60)
    # untrained: the loss of a uniform guess over 97 tokens or above
    assert r["first"] > 0.9 * math.log(ex.VOCAB)
    assert r["last"] < 0.5 * r["first"]
    assert r["greedy_is_best"] and r["chosen"] <= 0
