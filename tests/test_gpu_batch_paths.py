"""Paths of the batch operations that the shapes of test_gpu_batch.py do not
reach, against the same formulas in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import batch_reference as ref
from dolittle_amd import _lib
from dolittle_amd.batch import BatchShape, workspace_bytes
from test_gpu_batch import Problem, stored, value_of

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


def same_bits(a, b):
    return np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8))


# In BF16 16 or 32 rows in each wavefront with keys and values in LDS for all
# four (one and two row tiles), every width's tiles, whole and in pieces; in
# FP32 the form of few rows.  Few rows in both for the last two.
FORMS = [
    # batch, rows, prefix, capacity, (query heads, KV heads, width), lengths
    (2, 20, 70, 150, (8, 2, 128), [150, 67]),
    (1, 40, 37, 100, (4, 2, 64), [99]),
    (2, 20, 300, 90, (4, 1, 96), [90, 20]),
    (1, 20, 70, 90, (4, 1, 256), [77]),
    (1, 66, 8100, 70, (8, 8, 128), [69]),
    (1, 66, 0, 8200, (8, 8, 64), [200]),
    (1, 66, 0, 8200, (8, 8, 88), [131]),
    (2, 6, 40, 70, (4, 2, 128), [70, 41]),
    (2, 1, 40, 70, (4, 2, 96), [70, 41]),
]
forms = pytest.mark.parametrize("batch,rows,prefix,capacity,heads,lengths", FORMS)
types = pytest.mark.parametrize("dtype", ["bf16", "f32"])


def special_feature(oracle, dtype, rows, feature, value):
    """Those rows with one feature replaced."""
    rows = rows.copy()
    rows[..., feature] = stored(oracle, np.float32([value]), dtype)[0]
    return rows


@types
@forms
@pytest.mark.parametrize("special", [np.inf, -np.inf, np.nan])
def test_special_keys(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths, special):
    """A feature of a late new row's key is not finite and every query's is 1: a score of -inf is a key without
    weight, +inf and NaN make the rows that see it NaN, and rows that do not see it keep their bits."""
    feature, late = heads[2] // 2 + 1, min(rows, 2)
    p = Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths)
    p.q = special_feature(oracle, dtype, p.q, feature, 1.0)
    clean, _ = p.run(device, queue)
    keys = p.k.copy()
    for b, n in enumerate(lengths):
        p.k[b, n - late] = special_feature(oracle, dtype, p.k[b, n - late], feature, special)
    got, weights = p.run(device, queue)
    assert same_bits(got[:, :rows - late], clean[:, :rows - late])
    if special != -np.inf:
        assert np.all(np.isnan(value_of(got[:, rows - late:])))
        for b, n in enumerate(lengths):
            assert np.all(np.isnan(weights[b, :, :n])) and np.all(weights[b, :, n:] == -7.0)
        return
    # The late rows' formula without that key: every later key moves down by one.
    operands = [value_of(x) for x in (p.q, p.pk, p.pv, keys, p.v)]
    without = [x.copy() for x in operands]
    for b, n in enumerate(lengths):
        for x, full in zip(without[3:], operands[3:]):
            x[b, n - late:n - 1] = full[b, n - late + 1:n]
    fewer = [n - 1 for n in lengths]
    out, bound, _, _ = ref.attention(*without, fewer, float(p.scale), dtype)
    off = np.abs(value_of(got) - out)[:, rows - late:]
    assert np.all(off <= bound[:, rows - late:])
    # Weights: the earlier rows see their keys as they were, the late rows those of the shorter cache.
    early = [operands[0][:, :rows - late], *operands[1:]]
    _, _, first, first_bound = ref.attention(*early, [n - late for n in lengths], float(p.scale), dtype)
    tail = [operands[0][:, rows - late:], without[1], without[2], without[3], without[4]]
    _, _, last, last_bound = ref.attention(*tail, fewer, float(p.scale), dtype)
    for b, n in enumerate(lengths):
        assert np.array_equal(weights[b, :, n - late], p.weights[b, :, n - late])
        assert np.all(weights[b, :, n:] == -7.0)
        rest = [j for j in range(n) if j != n - late]
        added = first[b][:, rest] + last[b][:, :n - 1]
        total = p.weights[b][:, rest] + added
        wide = first_bound[b][:, rest] + last_bound[b][:, :n - 1] + 2.0 ** -23 * np.abs(total)
        wide += added * (rows * heads[0] // heads[1]) * 2.0 ** -24  # a rounding for each row and head added
        assert np.all(np.abs(weights[b][:, rest] - total) <= wide)
