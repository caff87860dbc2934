"""Paths of the batch operations that the shapes of test_gpu_batch.py do not
reach, against the same formulas in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from dolittle_amd import _lib
from dolittle_amd.batch import BatchShape, workspace_bytes
from test_gpu_batch import stored, value_of

pytestmark = pytest.mark.gpu


def test_caches_of_more_rows_than_32_bits_count(device, queue, oracle):
    """The last sequence's rows start at row 2^32: 16 caches of 2^28 slots lie before them."""
    batch, capacity, n = 17, 1 << 28, 3
    keys, values = (device.allocate(batch * capacity * 2) for _ in range(2))
    for sequence, rows in ((0, [10.0, 10.0, 10.0]), (batch - 1, [1.0, 2.0, 6.0])):
        queue.write(keys, np.zeros(n, np.uint16), sequence * capacity * 2)
        queue.write(values, stored(oracle, rows, "bf16"), sequence * capacity * 2)
    lengths = device.upload_array(queue, np.array([n] + [0] * (batch - 2) + [n], np.uint64))
    q = device.upload_array(queue, stored(oracle, np.ones(batch), "bf16"))
    out, scale = device.allocate(batch * 2), device.upload_array(queue, np.ones(1, np.float32))
    shape = BatchShape(batch, 1, 1, 1, 1, capacity)
    room = workspace_bytes("dl_attention_shared", shape, 0)
    work = device.allocate(room)
    _lib.call("dl_attention_shared", queue.handle, 1, C.byref(shape), q.ptr(), None, None, 0, keys.ptr(), values.ptr(),
              lengths.ptr(), out.ptr(), scale.ptr(), work.ptr(), room)
    got = value_of(queue.read(out, np.uint16, batch))
    # Equal scores: the mean of three values, exact in every step but the division.
    assert np.array_equal(got, [10.0] + [0.0] * (batch - 2) + [3.0])
