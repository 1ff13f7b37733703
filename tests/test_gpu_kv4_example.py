"""The serving example runs, returns its pages, and stays as near an uncompressed cache as 4 bits allow.

A group of 64 normal elements spans about 5 standard deviations, so a step is a
third of one and rounding adds step / sqrt(12), about 0.1 of each value, to
keys and values alike: between 0.01 (nothing is quantised away) and 0.3."""
from __future__ import annotations

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def test_serving_example(pkg):
    path = os.path.join(pkg.ROOT_DIR, "examples", "kv4_serving.py")
    spec = importlib.util.spec_from_file_location("kv4_serving", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    steps, difference = example.serve()
    assert steps > 12 and 0.01 < difference < 0.3
    with pytest.raises(RuntimeError):
        example.serve(pages=3)
