"""The example of a layer of experts: training with grouped products and
orthogonalised updates, serving on 4-bit weights."""
import importlib.util
import os

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_expert_layer_trains_and_serves():
    spec = importlib.util.spec_from_file_location("expert_layer", os.path.join(ROOT, "examples", "expert_layer.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, off = example.main(["--steps", "20", "--tokens", "300"])
    assert losses[-1] < 0.5 * losses[0]
    # weights of 4 bits are off by 1 / 12 of a 15th of their range, about 0.1 of
    # their size; three layers of them, each averaging over its inputs
    assert 0.0 < off < 0.5
