"""The hybrid example: training, prompts, forks, single tokens, trimming and compaction in one program."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_hybrid_example(gpu_lib):
    spec = importlib.util.spec_from_file_location("hybrid", os.path.join(ROOT, "examples", "hybrid.py"))
    hybrid = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(hybrid)
    # bf16 layers: each rounds its output once (2e-3 relative) and the served form sums in another order
    assert hybrid.main(T=150, steps=24, ways=2) < 1e-2
