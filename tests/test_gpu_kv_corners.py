"""Corner calls of the quantised key/value cache and window attention, against plain 64-bit
restatements. Tolerances are those of the ordinary cases unless a test derives its own."""
import ctypes

import pytest
import torch

import kv_ref as ref
from test_gpu_kv import DEV, DTYPES, close, gen, ints, kv, rows, starts, window_case  # noqa: F401 (kv: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f16", 64), ("bf16", 64), ("f16", 24), ("f32", 192)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 50])
def test_windows_near_the_largest_number(kv, dtype, dim, window):
    """A window that shows everything, with queries before the first key: their positions are negative."""
    window_case(kv, dtype, dim, 1, 2, [40, 3, 150, 70], [-10, -3, -100, 20], window, 3)
