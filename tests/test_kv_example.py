"""The example of a layer over the paged cache, at a small size."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest


def _example():
    path = Path(__file__).resolve().parent.parent / "examples" / "long_context.py"
    spec = importlib.util.spec_from_file_location("long_context", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.gpu
@pytest.mark.parametrize("chosen", [4, 40])
def test_example(chosen):
    got = _example().run(3, 1000, chosen, 5, heads=8, heads_kv=2, dim=64, chunk=384)
    assert got["finite"] and got["prompt_tokens_per_s"] > 0 and got["decode_us_per_step"] > 0
    share = got["weight_of_the_chosen"]
    if chosen == 40:  # every block: both sums are of the same weights (fp32 sums, log and exp)
        assert abs(share - 1.0) < 1e-4
    else:  # the best quarter of the blocks holds more than a tenth of the weight, and not all
        assert 0.1 < share < 1.0
