"""The fine-tuning example runs, learns its batch, and gives the same losses again."""
import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "finetune_step.py")


def test_example_learns_its_batch(rq, dev):
    spec = importlib.util.spec_from_file_location("finetune_step", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, norms = m.train(steps=12, report=lambda s: print(s, flush=True))
    assert all(map(math.isfinite, losses + norms)) and min(norms) > 0
    assert abs(losses[0] - math.log(512)) < 1.0      # a guess over the vocabulary
    assert losses[-1] < losses[0] - 0.5
