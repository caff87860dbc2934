"""Weights and caches held in 4 bits: mirror of the dl_fp4_* / dl_projection_fp4 /
dl_cache_append_fp4 / dl_attention_fp4 operations of include/dolittle_hip.h.

No counterpart in the reference, which keeps weights and caches in BF16 or FP32.
Results are within tolerance of the values that the 4 bits stand for; the
conforming operations are the catalog's dl_projection and dl_attention.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .batch import _CODES, BatchShape, _at
from .runtime import Device, DeviceBuffer, Queue

CacheAddresses = _lib.Fp4Cache


def row_bytes(rows: int, width: int) -> tuple[int, int]:
    """Bytes of the codes and of the scales of `rows` rows."""
    codes, scales = C.c_uint64(0), C.c_uint64(0)
    _lib.call("dl_fp4_bytes", rows, width, C.byref(codes), C.byref(scales))
    return codes.value, scales.value


def attention_workspace_bytes(shape: BatchShape, window: int = 0, sinks: int = 0) -> int:
    out = C.c_uint64(0)
    _lib.call("dl_attention_fp4_bytes", C.byref(shape), window, sinks, C.byref(out))
    return out.value


def _code(dtype: str) -> int:
    if dtype not in _CODES:
        raise _lib.InvalidArgument("unsupported storage type")
    return _CODES[dtype]


class Fp4Weight:
    """A weight [outputs][inputs] in 4 bits.  Every method only enqueues; operands are
    device addresses or buffers."""

    def __init__(self, device: Device, queue: Queue, outputs: int, inputs: int):
        codes, scales = row_bytes(outputs, inputs)
        self.queue, self.outputs, self.inputs = queue, outputs, inputs
        self.codes, self.scales = device.allocate(codes), device.allocate(scales)

    def quantize(self, weight, dtype: str = "bf16") -> None:
        """Takes the row-major weight's values."""
        _lib.call("dl_fp4_quantize", self.queue.handle, _code(dtype), _at(weight), self.codes.ptr(), self.scales.ptr(),
                  self.outputs, self.inputs)

    def values(self, output, dtype: str = "bf16") -> None:
        """The row-major values that the weight stands for."""
        _lib.call("dl_fp4_values", self.queue.handle, _code(dtype), self.codes.ptr(), self.scales.ptr(), _at(output),
                  self.outputs, self.inputs)

    def project(self, x, y, rows: int = 1, dtype: str = "bf16", output_position=None) -> None:
        """y [rows][outputs] = x [rows][inputs] times the weight; with an output position (a device word) the rows
        from that one on are written."""
        _lib.call("dl_projection_fp4", self.queue.handle, _code(dtype), _at(x), self.codes.ptr(), self.scales.ptr(), _at(y),
                  rows, self.inputs, self.outputs, _at(output_position))


class Fp4Cache:
    """The caches of `batch` sequences in 4 bits, read whole or through a sliding
    window with first rows that stay visible.  A window bounds what a step reads and not
    what the cache holds: `capacity` is for every row of a sequence.

    The host keeps each sequence's length, so a row that does not fit is refused
    here.  Every method only enqueues, except that a first attend that needs more
    workspace allocates it: run a step once before it is recorded into a graph.
    Recording a step counts its rows in `used` once; add those of every replay after
    the first.  `query` and the rows are device addresses or buffers,
    [batch][rows][heads][width].
    """

    def __init__(self, device: Device, queue: Queue, batch: int, capacity: int, query_heads: int, kv_heads: int,
                 width: int, dtype: str = "bf16", theta: float = 1e6, first_position: int = 0, window: int = 0,
                 sinks: int = 0):
        self._dtype = _code(dtype)
        if min(batch, capacity, query_heads, kv_heads, width) <= 0 or min(first_position, window, sinks) < 0:
            raise _lib.InvalidArgument("empty batch shape or negative window")
        self.device, self.queue, self.dtype, self.theta = device, queue, dtype, theta
        self.window, self.sinks = window, sinks
        self._dims = (query_heads, kv_heads, width)
        self.batch, self.capacity = batch, capacity
        codes, scales = row_bytes(batch * kv_heads * capacity, width)
        self._buffers = [device.allocate(n) for n in (codes, scales, codes, scales)]
        self.key_codes, self.key_scales, self.value_codes, self.value_scales = self._buffers
        self.addresses = CacheAddresses(*(b.ptr() for b in self._buffers))
        self.lengths = device.upload_array(queue, np.zeros(batch, np.uint64))
        self.positions = device.upload_array(queue, np.full(batch, first_position, np.uint64))
        self._scale = device.allocate(4)
        _lib.call("dl_attention_scale", queue.handle, self._scale.ptr(), width)
        self.used = [0] * batch
        self._work: list[DeviceBuffer] = []

    def shape(self, rows: int = 1) -> BatchShape:
        qh, kvh, w = self._dims
        return BatchShape(self.batch, rows, qh, kvh, w, self.capacity)

    def append(self, query, key, value, rotated, rows: int = 1) -> None:
        """New rows at each sequence's own length and position; `rotated` receives the rotated query."""
        if max(self.used) + rows > self.capacity:
            raise _lib.LengthError("new rows exceed the cache's capacity")
        shape = self.shape(rows)
        _lib.call("dl_cache_append_fp4", self.queue.handle, self._dtype, C.byref(shape), _at(query), _at(key), _at(value),
                  _at(rotated), C.byref(self.addresses), self.lengths.ptr(), self.lengths.ptr(), self.positions.ptr(),
                  self.positions.ptr(), self.theta)
        self.used = [n + rows for n in self.used]

    def attend(self, query, output, rows: int = 1) -> None:
        """Attention of the last `rows` rows."""
        shape = self.shape(rows)
        work, room = self._workspace(attention_workspace_bytes(shape, self.window, self.sinks))
        _lib.call("dl_attention_fp4", self.queue.handle, self._dtype, C.byref(shape), _at(query), C.byref(self.addresses),
                  self.lengths.ptr(), self.window, self.sinks, _at(output), self._scale.ptr(), work, room)

    def _workspace(self, need: int) -> tuple[C.c_void_p, int]:
        """One workspace for the queue's operations, which run in order.  Smaller ones that it outgrew are kept,
        for submitted and recorded work still uses them; each is at least twice the last."""
        if need and (not self._work or self._work[-1].nbytes < need):
            self._work.append(self.device.allocate(max(need, 2 * self._work[-1].nbytes if self._work else 0)))
        return (self._work[-1].ptr(), self._work[-1].nbytes) if self._work else (None, 0)
