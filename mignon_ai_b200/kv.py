"""The quantised key/value cache and the attention around it, on torch CUDA tensors.

For callers that run their own attention layers next to the engine (which keeps float32 rings of
its own):

* ``KvCache.write``      quantises rows of keys and values into a cache of 4 or 8 bits
* ``KvCache.read``       reads positions back as rows
* ``KvCache.attend``     one query token per session over its cached positions
* ``window_attention``   causal attention of whole segments, unquantised

All four share one mask: a query at position p sees the positions j <= p with j < sinks or
j > p - window (window 0: every one), as far as the cache still holds them. Rows are
``[rows, heads, head_dim]`` float32, float16 or bfloat16 tensors; ragged segments are given by int32
device tensors of their first rows (n + 1 of them). Calls go to the current stream of the tensors'
device, allocate at most their output and never synchronize. There is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import c_vp

_i = ctypes.c_int


class _Rows(ctypes.Structure):
    _fields_ = [("data", c_vp), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _Spec(ctypes.Structure):
    _fields_ = [(n, _i) for n in ("sessions", "heads", "head_dim", "bits", "slots", "sinks")]


_rows_p = ctypes.POINTER(_Rows)
_lib.register({
    "mc_kv_open": [_i, ctypes.POINTER(_Spec), ctypes.POINTER(c_vp)],
    "mc_kv_close": [c_vp],
    "mc_kv_error": [c_vp],
    "mc_kv_write_dev": [c_vp, _rows_p, _rows_p, _i, _i, c_vp, c_vp, c_vp, _i, c_vp],
    "mc_kv_read_dev": [c_vp, _rows_p, _rows_p, _i, _i, c_vp, c_vp, c_vp, c_vp, _i, c_vp],
    "mc_kv_attend_dev": [c_vp, _rows_p, _rows_p, _i, _i, c_vp, c_vp, _i, _i, ctypes.c_float, c_vp],
    "mc_window_attn_dev": [_rows_p, _rows_p, _rows_p, _rows_p] + [_i] * 6 + [c_vp, c_vp, _i, _i, _i, ctypes.c_float, c_vp],
})

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _check(name: str, x: torch.Tensor, device: torch.device, heads: Optional[int], dim: int,
           dtype: Optional[torch.dtype] = None):
    if x.dim() != 3 or x.shape[2] != dim or (heads is not None and x.shape[1] != heads):
        raise ValueError(f"{name}: expected [rows, {heads or 'heads'}, {dim}], got {tuple(x.shape)}")
    if x.dtype not in _DTYPES or (dtype is not None and x.dtype != dtype):
        raise TypeError(f"{name}: {x.dtype} (float32, float16 or bfloat16, the same in all tensors of a call)")
    if x.device != device:
        raise ValueError(f"{name}: on {x.device}, expected {device}")
    if dim > 1 and x.stride(2) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")


def _rows(x: torch.Tensor) -> _Rows:
    # an empty tensor has no address, and the library takes no null rows
    return _Rows(x.data_ptr() or 16, x.stride(0), x.stride(1))


def _ints(name: str, x: Optional[torch.Tensor], count: int, device: torch.device) -> Optional[int]:
    if x is None:
        return None
    if x.dtype != torch.int32 or x.device != device or x.dim() != 1 or x.shape[0] != count or not x.is_contiguous():
        raise ValueError(f"{name}: expected {count} contiguous int32 on {device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.data_ptr()


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class KvCache:
    """Keys and values of ``sessions`` sessions of one attention layer, held in 4 or 8 bits.

    A session keeps its first ``sinks`` positions and the last ``slots - sinks``. Close it (or let
    it go) when its work is done: ``close`` waits for the device.
    """

    def __init__(self, sessions: int, heads: int, head_dim: int, slots: int, bits: int = 4, sinks: int = 0, device: int = 0):
        self._h = c_vp()
        spec = _Spec(sessions, heads, head_dim, bits, slots, sinks)
        _lib.check(_lib.lib().mc_kv_open(device, ctypes.byref(spec), ctypes.byref(self._h)))
        self.sessions, self.heads, self.head_dim, self.slots = sessions, heads, head_dim, slots
        self.bits, self.sinks, self.device = bits, sinks, torch.device("cuda", device)

    def close(self):
        if self._h:
            h, self._h = self._h, c_vp()
            _lib.check(_lib.lib().mc_kv_close(h))

    def __del__(self):
        try:
            if getattr(self, "_h", None):
                _lib.lib().mc_kv_close(self._h)
                self._h = c_vp()
        except Exception:  # interpreter shutdown
            pass

    def check(self):
        """Waits for the device and raises if a call named a session or position out of range."""
        _lib.check(_lib.lib().mc_kv_error(self._h))

    def _segments(self, n_rows, pos0, row_start, sessions):
        n = pos0.shape[0]
        if row_start is None and n != n_rows:
            raise ValueError(f"without row_start every row is a segment: {n_rows} rows, {n} positions")
        return (_ints("row_start", row_start, n + 1, self.device), _ints("sessions", sessions, n, self.device),
                _ints("pos0", pos0, n, self.device), n)

    def write(self, k: torch.Tensor, v: torch.Tensor, pos0: torch.Tensor, row_start: Optional[torch.Tensor] = None,
              sessions: Optional[torch.Tensor] = None):
        """Quantises rows into the cache: rows [row_start[b], row_start[b+1]) of k and v are
        positions pos0[b], pos0[b]+1, ... of session sessions[b] (default b). Without row_start
        every row is a segment of its own, as in a decode step."""
        _check("k", k, self.device, self.heads, self.head_dim)
        _check("v", v, self.device, self.heads, self.head_dim, k.dtype)
        if v.shape[0] != k.shape[0]:
            raise ValueError(f"k has {k.shape[0]} rows, v {v.shape[0]}")
        start, sess, pos, n = self._segments(k.shape[0], pos0, row_start, sessions)
        _lib.check(_lib.lib().mc_kv_write_dev(self._h, _rows(k), _rows(v), _DTYPES[k.dtype], k.shape[0], start, sess, pos,
                                              n, _stream(self.device)))

    def read(self, pos0: torch.Tensor, lens: torch.Tensor, row_start: Optional[torch.Tensor] = None,
             n_rows: Optional[int] = None, sessions: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float32,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Reads positions back: rows [row_start[b], row_start[b+1]) are positions pos0[b], ... of a
        session that has lens[b] positions so far; those not held, and rows of no segment, are zeros. n_rows is row_start's
        last entry (row_start is on the device); not needed with `out` or without row_start."""
        if out is None:
            if n_rows is None:
                if row_start is not None:
                    raise ValueError("read: give n_rows (the last entry of row_start) or out")
                n_rows = pos0.shape[0]
            out = tuple(torch.empty((n_rows, self.heads, self.head_dim), dtype=dtype, device=self.device) for _ in range(2))
        k, v = out
        _check("out[0]", k, self.device, self.heads, self.head_dim)
        _check("out[1]", v, self.device, self.heads, self.head_dim, k.dtype)
        if v.shape[0] != k.shape[0]:
            raise ValueError(f"out: {k.shape[0]} and {v.shape[0]} rows")
        start, sess, pos, n = self._segments(k.shape[0], pos0, row_start, sessions)
        _lib.check(_lib.lib().mc_kv_read_dev(self._h, _rows(k), _rows(v), _DTYPES[k.dtype], k.shape[0], start, sess, pos,
                                             _ints("lens", lens, n, self.device), n, _stream(self.device)))
        return k, v

    def attend(self, q: torch.Tensor, lens: torch.Tensor, sessions: Optional[torch.Tensor] = None, window: int = 0,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of one query token per session: row i of q [n, q_heads, head_dim] belongs to
        session sessions[i] (default i), which has lens[i] positions, the query's own the last.
        scale defaults to 1 / sqrt(head_dim)."""
        _check("q", q, self.device, None, self.head_dim)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        else:
            _check("out", out, self.device, q.shape[1], self.head_dim, q.dtype)
            if out.shape[0] != q.shape[0]:
                raise ValueError(f"out has {out.shape[0]} rows, q {q.shape[0]}")
        n = q.shape[0]
        _lib.check(_lib.lib().mc_kv_attend_dev(
            self._h, _rows(q), _rows(out), _DTYPES[q.dtype], q.shape[1], _ints("sessions", sessions, n, self.device),
            _ints("lens", lens, n, self.device), n, window, 1 / math.sqrt(self.head_dim) if scale is None else scale,
            _stream(self.device)))
        return out


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_start: Optional[torch.Tensor] = None,
                     k_start: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of ragged segments: queries [q_start[b], q_start[b+1]) of q [rows, q_heads,
    head_dim] over keys [k_start[b], k_start[b+1]) of k and v [rows, heads, head_dim]. A segment's
    queries are its last positions (k_start defaults to q_start; both None: one segment). A row
    that sees nothing is zero; rows of no segment are not written."""
    device, dim = q.device, q.shape[-1]
    if device.type != "cuda":
        raise ValueError("q: expected a CUDA tensor")
    _check("q", q, device, None, dim)
    _check("k", k, device, None, dim, q.dtype)
    _check("v", v, device, k.shape[1], dim, q.dtype)
    if v.shape[0] != k.shape[0]:
        raise ValueError(f"k has {k.shape[0]} rows, v {v.shape[0]}")
    if q_start is None and k_start is not None:
        raise ValueError("k_start without q_start")
    if k_start is None:
        k_start = q_start
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    else:
        _check("out", out, device, q.shape[1], dim, q.dtype)
        if out.shape[0] != q.shape[0]:
            raise ValueError(f"out has {out.shape[0]} rows, q {q.shape[0]}")
    n = 1 if q_start is None else q_start.shape[0] - 1
    with torch.cuda.device(device):
        _lib.check(_lib.lib().mc_window_attn_dev(
            _rows(q), _rows(k), _rows(v), _rows(out), _DTYPES[q.dtype], q.shape[1], k.shape[1], dim, q.shape[0], k.shape[0],
            _ints("q_start", q_start, n + 1, device), _ints("k_start", k_start, n + 1, device), n, window, sinks,
            1 / math.sqrt(dim) if scale is None else scale, _stream(device)))
    return out
