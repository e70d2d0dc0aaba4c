"""The example runs as it is written down: it learns, and a beam search's scores are those of its sequences."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_beam_search_example():
    spec = importlib.util.spec_from_file_location("beam_search_example", os.path.join(ROOT, "examples", "beam_search.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    first, last, off = example.main(steps=30, beams=3, new=8)
    assert last < 0.9 * first
    # float models: 8 scores of about 1, each a sum over float products in another order (chunks there, single tokens here)
    assert off < 1e-3
