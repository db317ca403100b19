"""The example that serves attention layers from the quantised cache: its calls, one after the other,
against one plain float32 pass over the same rows."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "quantised_cache.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("quantised_cache", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


# A row's codes are off by at most half a step: for normal rows of 64 values, whose extremes lie about
# 2.4 deviations out, uniform errors of 2.4/15 (4 bits) or 2.4/127/2 (8 bits), so 0.09 or 0.006 of a
# value's deviation; attention averages them over its keys, and two residual layers pass on at most what
# they add. bfloat16's rounding of every product's inputs and outputs adds about 0.005.
@pytest.mark.parametrize("bits,most", [(4, 0.10), (8, 0.02)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_second_prompts_are_near_the_float32_ones(example, bits, most, window, sinks):
    got, want, _ = example.run(sessions=9, bits=bits, window=window, sinks=sinks, prompt_rows=70, steps=5, second=11)
    off = ((got[:len(want)].float() - want).norm() / want.norm()).item()
    assert off <= most
