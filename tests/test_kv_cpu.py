"""What the cache's entry points refuse, which needs no device: every check comes before the first
CUDA call."""
import ctypes

import pytest

from mignon_ai_b200 import _lib, kv

INVALID = 1


def spec(**c):
    d = dict(sessions=2, heads=2, head_dim=64, bits=4, slots=100, sinks=4)
    d.update(c)
    return kv._Spec(*(d[n] for n, _ in kv._Spec._fields_))


@pytest.mark.parametrize("bad", [dict(sessions=0), dict(heads=0), dict(head_dim=0), dict(head_dim=24), dict(head_dim=144),
                                 dict(bits=2), dict(bits=16), dict(slots=0), dict(sinks=-1), dict(sinks=100),
                                 dict(slots=(1 << 30) + 1)])
def test_open_refuses(bad):
    h = ctypes.c_void_p()
    assert _lib.lib().mc_kv_open(0, ctypes.byref(spec(**bad)), None, None, ctypes.byref(h)) == INVALID
    assert _lib.lib().mc_last_error() and not h
    n = ctypes.c_size_t()
    assert _lib.lib().mc_kv_bytes(ctypes.byref(spec(**bad)), ctypes.byref(n)) == INVALID


def test_bytes():
    """Codes of 4 or 8 bits and two 16-bit numbers a row, slots rounded up to 64, and the workspace."""
    for bits, dim, slots in ((4, 64, 100), (8, 128, 64), (4, 16, 1)):
        n = ctypes.c_size_t()
        assert _lib.lib().mc_kv_bytes(ctypes.byref(spec(bits=bits, head_dim=dim, slots=slots, sinks=0)), ctypes.byref(n)) == 0
        rows = 2 * 2 * 2 * ((slots + 63) // 64 * 64)
        assert 0 <= n.value - rows * (dim * bits // 8 + 4) <= 12 << 20
    assert _lib.lib().mc_kv_open(0, ctypes.byref(spec()), 100, None, ctypes.byref(ctypes.c_void_p())) == INVALID  # not aligned


def test_null_arguments():
    L = _lib.lib()
    h = ctypes.c_void_p()
    assert L.mc_kv_open(0, None, None, None, ctypes.byref(h)) == INVALID
    assert L.mc_kv_open(0, ctypes.byref(spec()), None, None, None) == INVALID
    assert L.mc_kv_bytes(None, None) == INVALID
    assert L.mc_kv_error(None) == INVALID
    assert L.mc_kv_close(None) == 0
    r = ctypes.byref(kv._Rows(16, 64, 64))
    assert L.mc_kv_write_dev(None, r, r, 0, 1, None, None, 16, 1, None) == INVALID
    assert L.mc_kv_read_dev(None, r, r, 0, 1, None, None, 16, 16, 1, None) == INVALID
    assert L.mc_kv_attend_dev(None, r, r, 0, 2, None, 16, 1, 0, 1.0, None) == INVALID


WINDOW = dict(dtype=0, q_heads=4, kv_heads=2, head_dim=64, n_q=5, n_k=5, q_start=None, k_start=None, n_segments=1,
              window=0, sinks=0, scale=1.0)


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dtype=-1), dict(q_heads=3), dict(q_heads=0), dict(kv_heads=0),
                                 dict(head_dim=0), dict(head_dim=257), dict(n_q=-1), dict(n_k=-1), dict(n_segments=2),
                                 dict(q_start=16), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
                                 dict(scale=float("inf")), dict(scale=float("nan"))])
def test_window_refuses(bad):
    r = ctypes.byref(kv._Rows(16, 64, 64))
    args = list({**WINDOW, **bad}.values())
    assert _lib.lib().mc_window_attn_dev(r, r, r, r, *args, None) == INVALID
    assert _lib.lib().mc_last_error()


def test_window_takes_no_null_rows_and_nothing_to_do():
    r, null = ctypes.byref(kv._Rows(16, 64, 64)), ctypes.byref(kv._Rows(None, 64, 64))
    assert _lib.lib().mc_window_attn_dev(null, r, r, r, *WINDOW.values(), None) == INVALID
    assert _lib.lib().mc_window_attn_dev(r, r, r, r, *{**WINDOW, "n_q": 0}.values(), None) == 0
