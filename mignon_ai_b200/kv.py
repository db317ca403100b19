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
device, allocate at most their output and never synchronize; ``KvCache.check`` and ``check`` do, and
raise what the kernels found. There is no CPU path.
"""
from __future__ import annotations

import ctypes
import struct
import threading
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import c_vp

_i = ctypes.c_int


class _Rows(ctypes.Structure):
    _fields_ = [("data", c_vp), ("row_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64)]


class _Spec(ctypes.Structure):
    _fields_ = [(n, _i) for n in ("sessions", "heads", "head_dim", "bits", "slots", "sinks")]


_lib.register({
    "mc_kv_bytes": [ctypes.POINTER(_Spec), ctypes.POINTER(ctypes.c_size_t)],
    "mc_kv_open": [_i, ctypes.POINTER(_Spec), c_vp, c_vp, ctypes.POINTER(c_vp)],
    "mc_kv_close": [c_vp],
    "mc_kv_error": [c_vp],
    "mc_window_error": [_i],
    "mc_kv_write_dev": [c_vp, c_vp, c_vp, _i, _i, c_vp, c_vp, c_vp, _i, c_vp],
    "mc_kv_read_dev": [c_vp, c_vp, c_vp, _i, _i, c_vp, c_vp, c_vp, c_vp, _i, c_vp],
    "mc_kv_attend_dev": [c_vp, c_vp, c_vp, _i, _i, c_vp, c_vp, _i, _i, ctypes.c_float, c_vp],
    "mc_window_attn_dev": [c_vp, c_vp, c_vp, c_vp] + [_i] * 6 + [c_vp, c_vp, _i, _i, _i, ctypes.c_float, c_vp],
})

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


_raw_stream = torch._C._cuda_getCurrentRawStream
_pack = struct.Struct("12q").pack_into  # up to four mc_rows


class _Scratch(threading.local):
    """The mc_rows of a call (a thread's own: the library reads them while the GIL is released)."""

    def __init__(self):
        self.buf = ctypes.create_string_buffer(4 * ctypes.sizeof(_Rows))
        at = ctypes.addressof(self.buf)
        self.rows = tuple(at + i * ctypes.sizeof(_Rows) for i in range(4))


_scratch = _Scratch()


def _rows(name: str, x: torch.Tensor, index: int, heads: Optional[int], dim: int, dtype: torch.dtype,
          count: Optional[int] = None) -> Tuple[int, int, int]:
    """Address, row stride and head stride of rows [count, heads, dim] on device `index`."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != dim or (heads is not None and shape[1] != heads) or (
            count is not None and shape[0] != count):
        raise ValueError(f"{name}: expected [{'rows' if count is None else count}, {heads or 'heads'}, {dim}], got {tuple(shape)}")
    if shape[0] >> 31 or shape[1] >> 31:
        raise ValueError(f"{name}: {tuple(shape)} does not fit 32 bits")
    if x.dtype is not dtype:
        raise TypeError(f"{name}: {x.dtype}, expected {dtype}")
    if x.get_device() != index:
        raise ValueError(f"{name}: on {x.device}, expected cuda:{index}")
    if stride[2] != 1 and dim > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    # an empty tensor has no address, and the library takes no null rows
    return x.data_ptr() or 16, stride[0], stride[1]


def _output(q: torch.Tensor) -> torch.Tensor:
    """Rows of q's shape, in q's order of strides unless q's rows overlap (then the last dimension's would
    not be 1)."""
    out = torch.empty_like(q)
    return out if out.stride(2) == 1 else torch.empty_like(q, memory_format=torch.contiguous_format)


def _address(x: torch.Tensor) -> Tuple[int, int, int]:
    """_rows of a tensor that was made here."""
    stride = x.stride()
    return x.data_ptr() or 16, stride[0], stride[1]


def _int32(name: str, x: int) -> int:
    """x, which ctypes would cut to 32 bits."""
    if not -2 ** 31 <= x < 2 ** 31:
        raise ValueError(f"{name}: {x} does not fit 32 bits")
    return x


def _dtype(x: torch.Tensor) -> int:
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"{x.dtype}: float32, float16 or bfloat16 rows are supported")
    return code


def _ints(name: str, x: Optional[torch.Tensor], count: int, index: int) -> Optional[int]:
    if x is None:
        return None
    if x.dtype is not torch.int32 or x.get_device() != index or x.shape != (count,) or not x.is_contiguous():
        raise ValueError(f"{name}: expected {count} contiguous int32 on cuda:{index}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.data_ptr() or 16  # as in _rows: null would mean that none were given


class KvCache:
    """Keys and values of ``sessions`` sessions of one attention layer, held in 4 or 8 bits.

    A session keeps its first ``sinks`` positions and the last ``slots - sinks``. The cache lies in
    ``memory``, a uint8 tensor allocated on the current stream; as with any tensor, work on other
    streams has to be done, or recorded on it, before the cache is closed or let go.
    """

    def __init__(self, sessions: int, heads: int, head_dim: int, slots: int, bits: int = 4, sinks: int = 0, device: int = 0):
        self._h = c_vp()
        numbers = dict(sessions=sessions, heads=heads, head_dim=head_dim, bits=bits, slots=slots, sinks=sinks)
        spec, n = _Spec(**{name: _int32(name, x) for name, x in numbers.items()}), ctypes.c_size_t()
        lib = _lib.lib()
        _lib.check(lib.mc_kv_bytes(ctypes.byref(spec), ctypes.byref(n)))
        self.memory = torch.empty(n.value, dtype=torch.uint8, device=torch.device("cuda", device))
        _lib.check(lib.mc_kv_open(device, ctypes.byref(spec), self.memory.data_ptr(), _raw_stream(device), ctypes.byref(self._h)))
        self.sessions, self.heads, self.head_dim, self.slots = sessions, heads, head_dim, slots
        self.bits, self.sinks, self.device = bits, sinks, torch.device("cuda", device)
        self._lib, self._index, self._scale = _lib.lib(), device, head_dim ** -0.5

    def close(self):
        if self._h:
            h, self._h, self.memory = self._h, c_vp(), None
            _lib.check(_lib.lib().mc_kv_close(h))

    def __del__(self):
        try:
            if getattr(self, "_h", None):
                _lib.lib().mc_kv_close(self._h)
                self._h = c_vp()
        except Exception:  # interpreter shutdown
            pass

    def check(self):
        """Waits for the device and raises if a call named a session, a position or a segment out of range,
        or a kernel gave up a wait."""
        _lib.check(_lib.lib().mc_kv_error(self._h))

    def _segments(self, n_rows, pos0, row_start, sessions):
        n = pos0.shape[0]
        if row_start is None and n != n_rows:
            raise ValueError(f"without row_start every row is a segment: {n_rows} rows, {n} positions")
        i = self._index
        return _ints("row_start", row_start, n + 1, i), _ints("sessions", sessions, n, i), _ints("pos0", pos0, n, i), n

    def write(self, k: torch.Tensor, v: torch.Tensor, pos0: torch.Tensor, row_start: Optional[torch.Tensor] = None,
              sessions: Optional[torch.Tensor] = None):
        """Quantises rows into the cache: rows [row_start[b], row_start[b+1]) of k and v are
        positions pos0[b], pos0[b]+1, ... of session sessions[b] (default b). Without row_start
        every row is a segment of its own, as in a decode step."""
        code, n_rows, index, s = _dtype(k), k.shape[0], self._index, _scratch
        _pack(s.buf, 0, *_rows("k", k, index, self.heads, self.head_dim, k.dtype),
              *_rows("v", v, index, self.heads, self.head_dim, k.dtype, n_rows), 0, 0, 0, 0, 0, 0)
        start, sess, pos, n = self._segments(n_rows, pos0, row_start, sessions)
        status = self._lib.mc_kv_write_dev(self._h, s.rows[0], s.rows[1], code, n_rows, start, sess, pos, n,
                                           _raw_stream(index))
        if status:
            _lib.check(status)

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
            k = torch.empty((n_rows, self.heads, self.head_dim), dtype=dtype, device=self.device)
            v = torch.empty_like(k)
            k_rows, v_rows = _address(k), _address(v)
        else:
            k, v = out
            n_rows = k.shape[0]
            k_rows = _rows("out[0]", k, self._index, self.heads, self.head_dim, k.dtype)
            v_rows = _rows("out[1]", v, self._index, self.heads, self.head_dim, k.dtype, n_rows)
        code, index, s = _dtype(k), self._index, _scratch
        _pack(s.buf, 0, *k_rows, *v_rows, 0, 0, 0, 0, 0, 0)
        start, sess, pos, n = self._segments(n_rows, pos0, row_start, sessions)
        status = self._lib.mc_kv_read_dev(self._h, s.rows[0], s.rows[1], code, n_rows, start, sess, pos,
                                          _ints("lens", lens, n, index), n, _raw_stream(index))
        if status:
            _lib.check(status)
        return k, v

    def attend(self, q: torch.Tensor, lens: torch.Tensor, sessions: Optional[torch.Tensor] = None, window: int = 0,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of one query token per session: row i of q [n, q_heads, head_dim] belongs to
        session sessions[i] (default i), which has lens[i] positions, the query's own the last.
        scale defaults to 1 / sqrt(head_dim)."""
        code, index, s = _dtype(q), self._index, _scratch
        rows = _rows("q", q, index, None, self.head_dim, q.dtype)
        n, q_heads, _ = q.shape
        if out is None:
            out = _output(q)
            out_rows = _address(out)
        else:
            out_rows = _rows("out", out, index, q_heads, self.head_dim, q.dtype, n)
        _pack(s.buf, 0, *rows, *out_rows, 0, 0, 0, 0, 0, 0)
        status = self._lib.mc_kv_attend_dev(
            self._h, s.rows[0], s.rows[1], code, q_heads, _ints("sessions", sessions, n, index),
            _ints("lens", lens, n, index), n, _int32("window", window), self._scale if scale is None else scale, _raw_stream(index))
        if status:
            _lib.check(status)
        return out


def check(device: Optional[int] = None):
    """Waits for the device (default: the current one) and raises if ``window_attention`` was given a
    segment out of range there, or a kernel of this module gave up a wait, since the last check."""
    _lib.check(_lib.lib().mc_window_error(torch.cuda.current_device() if device is None else device))


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_start: Optional[torch.Tensor] = None,
                     k_start: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of ragged segments: queries [q_start[b], q_start[b+1]) of q [rows, q_heads,
    head_dim] over keys [k_start[b], k_start[b+1]) of k and v [rows, heads, head_dim]. A segment's
    queries are its last positions (k_start defaults to q_start; both None: one segment). A row
    that sees nothing is zero; rows of no segment are not written, nor those of a segment out of
    range, which ``check`` reports."""
    index, dim, dtype, s = q.get_device(), q.shape[-1], q.dtype, _scratch
    if index < 0:
        raise ValueError("q: expected a CUDA tensor")
    code = _dtype(q)
    q_rows, k_rows = _rows("q", q, index, None, dim, dtype), _rows("k", k, index, None, dim, dtype)
    n_q, q_heads, _ = q.shape
    n_k, heads, _ = k.shape
    if out is None:
        out = _output(q)
        out_rows = _address(out)
    else:
        out_rows = _rows("out", out, index, q_heads, dim, dtype, n_q)
    _pack(s.buf, 0, *q_rows, *k_rows, *_rows("v", v, index, heads, dim, dtype, n_k), *out_rows)
    if k_start is None:
        k_start = q_start
    elif q_start is None:
        raise ValueError("k_start without q_start")
    n = 1 if q_start is None else q_start.shape[0] - 1
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return window_attention(q, k, v, q_start, k_start, window, sinks, scale, out)
    status = _lib.lib().mc_window_attn_dev(
        *s.rows, code, q_heads, heads, dim, n_q, n_k, _ints("q_start", q_start, n + 1, index),
        _ints("k_start", k_start, n + 1, index), n, _int32("window", window), _int32("sinks", sinks),
        dim ** -0.5 if scale is None else scale, _raw_stream(index))
    if status:
        _lib.check(status)
    return out
