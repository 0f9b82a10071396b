"""The serving operators together: examples/serve_block.py against attention without a cache."""
from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "serve_block.py"
    spec = importlib.util.spec_from_file_location("serve_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_serving_loop_matches_attention_without_a_cache(device):
    """Outputs are means of values of size 1 to 4 in bf16: they and the values are each off by up to 2^-8 of
    themselves, and projections of differently shaped batches may round the last bit of q, k and v otherwise."""
    lines = []
    worst = _example().serve(steps=24, check=True, say=lines.append)
    assert worst < 0.06, worst
    assert "forks" in lines[-1] and " 0 forks" not in lines[-1]
