"""A batch of sequences over a prefix that they share and bounded caches of
their own: mirror of the dl_attention_shared / dl_attention_weighted /
dl_cache_* operations of include/dolittle_hip.h.

No counterpart in the reference, whose cache is one contiguous sequence
(src/inference/cache/contiguous.cpp).  Results are within tolerance, not
bit-exact: the conforming attention is the catalog's dl_attention.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .runtime import Device, DeviceBuffer, Queue

BatchShape = _lib.BatchShape
_CODES = {"bf16": 1, "f32": 2}
_BYTES = {"bf16": 2, "f32": 4}


def workspace_bytes(operation: str, shape: BatchShape, argument: int) -> int:
    """Workspace of dl_attention_shared or dl_attention_weighted over a prefix
    of `argument` keys, or of dl_cache_evict to a budget of `argument` rows."""
    out = C.c_uint64(0)
    _lib.call(operation + "_bytes", C.byref(shape), argument, C.byref(out))
    return out.value


class BatchCache:
    """The caches of `batch` sequences that continue one prefix: keys, values,
    positions and accumulated weights on the device.

    The host keeps each sequence's length (append and evict change them by rules
    that need no device value), so a row that does not fit is refused here.
    Every method only enqueues, except that a first attend or evict that needs
    more workspace allocates it: run a step once before it is recorded into a
    graph.  Recording a step counts its rows in `used` once; add those of every
    replay after the first.  `query` and the rows are device addresses or
    buffers, [batch][rows][heads][width].
    """

    def __init__(self, device: Device, queue: Queue, batch: int, capacity: int, query_heads: int, kv_heads: int,
                 width: int, dtype: str = "bf16", theta: float = 1e6, first_position: int = 0):
        if dtype not in _CODES:
            raise _lib.InvalidArgument("unsupported storage type")
        if min(batch, capacity, query_heads, kv_heads, width) <= 0 or first_position < 0:
            raise _lib.InvalidArgument("empty batch shape")
        self.device, self.queue, self.dtype, self.theta = device, queue, dtype, theta
        self._dims = (query_heads, kv_heads, width)
        self.batch, self.capacity = batch, capacity
        rows = batch * capacity * kv_heads * width * _BYTES[dtype]
        self.keys, self.values = device.allocate(rows), device.allocate(rows)
        self.slots = device.allocate(batch * kv_heads * capacity * 4)
        self.weights = device.allocate(batch * kv_heads * capacity * 4)
        self.lengths = device.upload_array(queue, np.zeros(batch, np.uint64))
        self.positions = device.upload_array(queue, np.full(batch, first_position, np.uint64))
        self._scale = device.allocate(4)
        _lib.call("dl_attention_scale", queue.handle, self._scale.ptr(), width)
        self.used = [0] * batch
        self._prefix = (None, None, 0)
        self._work: list[DeviceBuffer] = []

    def shape(self, rows: int = 1) -> BatchShape:
        qh, kvh, w = self._dims
        return BatchShape(self.batch, rows, qh, kvh, w, self.capacity)

    def set_prefix(self, key, value, count: int) -> None:
        """The shared prefix's rotated keys and its values, [count][kv_heads][width]; borrowed."""
        self._prefix = (key, value, count) if count else (None, None, 0)

    def append(self, query, key, value, rotated, rows: int = 1) -> None:
        """New rows at each sequence's own length and position; `rotated` receives the rotated query."""
        if max(self.used) + rows > self.capacity:
            raise _lib.LengthError("new rows exceed the cache's capacity")
        shape = self.shape(rows)
        _lib.call("dl_cache_append", self.queue.handle, _CODES[self.dtype], C.byref(shape), _at(query), _at(key),
                  _at(value), _at(rotated), self.keys.ptr(), self.values.ptr(), self.lengths.ptr(), self.lengths.ptr(),
                  self.positions.ptr(), self.positions.ptr(), self.slots.ptr(), self.weights.ptr(), self.theta)
        self.used = [n + rows for n in self.used]

    def attend(self, query, output, rows: int = 1, accumulate: bool = True) -> None:
        """Attention of the last `rows` rows; with `accumulate` the weight each cached row received is added up."""
        name = "dl_attention_weighted" if accumulate else "dl_attention_shared"
        shape, (pk, pv, count) = self.shape(rows), self._prefix
        work, room = self._workspace(workspace_bytes(name, shape, count))
        weights = (self.weights.ptr(), self.weights.ptr()) if accumulate else ()
        _lib.call(name, self.queue.handle, _CODES[self.dtype], C.byref(shape), _at(query), _at(pk), _at(pv), count,
                  self.keys.ptr(), self.values.ptr(), self.lengths.ptr(), *weights, _at(output), self._scale.ptr(), work,
                  room)

    def evict(self, budget: int, sinks: int = 0, recent: int = 0) -> None:
        """Cuts every sequence to at most `budget` rows, keeping those at a position below `sinks`, the last `recent`
        and then the rows that received most attention.  Positions count from the sequence's start: behind a prefix
        of `sinks` or more positions, which holds those rows and is never cut, no own row is a sink."""
        if budget <= 0 or sinks < 0 or recent < 0:
            raise _lib.InvalidArgument("invalid eviction budget")
        shape = self.shape()
        work, room = self._workspace(workspace_bytes("dl_cache_evict", shape, budget))
        _lib.call("dl_cache_evict", self.queue.handle, _CODES[self.dtype], C.byref(shape), self.keys.ptr(),
                  self.values.ptr(), self.lengths.ptr(), self.lengths.ptr(), self.slots.ptr(), self.slots.ptr(),
                  self.weights.ptr(), self.weights.ptr(), budget, sinks, recent, work, room)
        self.used = [min(n, budget) for n in self.used]

    def _workspace(self, need: int) -> tuple[C.c_void_p, int]:
        """One workspace for the queue's operations, which run in order.  Smaller ones that it outgrew are kept,
        for submitted and recorded work still uses them; each is at least twice the last."""
        if not self._work or self._work[-1].nbytes < need:
            self._work.append(self.device.allocate(max(need, 2 * self._work[-1].nbytes if self._work else 0)))
        return self._work[-1].ptr(), self._work[-1].nbytes


def _at(operand):
    """A device address from a buffer, an address or None."""
    if operand is None:
        return None
    return operand.ptr() if isinstance(operand, DeviceBuffer) else C.c_void_p(int(operand))
