"""The bounded-cache example runs and keeps its sequences within their budget."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_bounded_cache_example(mb, torch_cuda):
    spec = importlib.util.spec_from_file_location(
        "bounded_cache", os.path.join(ROOT, "examples", "bounded_cache.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    lens, out = ex.main(steps=12, budget=96, recent=16, prompts=(90, 200, 5), every=4)
    assert lens == [96, 96, 17] and bool(torch_cuda.isfinite(out).all())
