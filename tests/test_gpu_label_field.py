"""The label operators together, as examples/label_field.py uses them: traced cells, their
rows, distillation and answers.  A field that has learned nothing has the loss of its first
step, log probabilities near -log(labels) and finds the best label of 128 by chance."""

import importlib.util
import math
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_label_field_learns():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    spec = importlib.util.spec_from_file_location(
        "label_field", os.path.join(ROOT, "examples", "label_field.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(points=6000, labels=128, features=16, size=64, cameras=6, batch=4096,
                     steps=40, log=lambda s: print(s, flush=True))
    assert all(math.isfinite(x) for x in r["loss"])
    assert sum(r["loss"][-5:]) < 0.5 * sum(r["loss"][:5])
    assert r["log_prob"] > -math.log(128) + 1.0
    assert r["first"] > 0.2 and r["in_five"] > 0.4
    assert 0.0 < r["entropy"] < math.log(128)
