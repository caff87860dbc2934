"""Paths of the batch operations that the shapes of test_gpu_batch.py do not
reach, against the same formulas in 64 bits."""
import ctypes as C

import numpy as np
import pytest

import batch_reference as ref
from dolittle_amd import _lib
from dolittle_amd.batch import BatchCache, BatchShape, workspace_bytes
from test_gpu_batch import CODE, Problem, evict_inputs, stored, up, value_of, want_evict

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


@types
@forms
def test_maxima_that_rise_in_many_steps(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths):
    """Keys that grow along the sources: scores of some hundreds, most rows' maximum in a late step, and what
    was summed before it is scaled down more than once."""
    p = Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths, spread=4.0)
    grow = lambda k, axis: stored(oracle, value_of(k) * np.linspace(0.1, 2.0, k.shape[axis]).reshape(  # noqa: E731
        [-1 if a == axis else 1 for a in range(k.ndim)]), dtype)
    p.pk = grow(p.pk, 0)
    for b, n in enumerate(lengths):
        p.k[b, :n] = grow(p.k[b, :n], 0)
    p.check(device, queue)


@types
@forms
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_scales(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths, scale):
    p = Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths)
    p.scale = np.float32(scale)
    p.check(device, queue)


@types
@forms
def test_zero_scale_with_an_infinite_key(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths):
    """0 * inf is NaN for the last new row, which sees the key, and nothing to the others."""
    p = Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths)
    p.scale = np.float32(0.0)
    clean, _ = p.run(device, queue)
    for b, n in enumerate(lengths):
        p.k[b, n - 1] = stored(oracle, np.full(heads[2], np.inf), dtype)
    got, weights = p.run(device, queue)
    assert same_bits(got[:, :-1], clean[:, :-1])
    assert np.all(np.isnan(value_of(got[:, -1])))
    for b, n in enumerate(lengths):
        assert np.all(np.isnan(weights[b, :, :n])) and np.all(weights[b, :, n:] == -7.0)


def special_feature(oracle, dtype, rows, feature, value):
    """Those rows with one feature replaced."""
    rows = rows.copy()
    rows[..., feature] = stored(oracle, np.float32([value]), dtype)[0]
    return rows


@types
@forms
@pytest.mark.parametrize("special", [np.inf, -np.inf, np.nan])
def test_special_values_stay_in_their_feature(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths,
                                              special):
    """One feature of the values of the last new rows, and of a late prefix row, is not finite: it reaches that
    feature of the rows that see it, and no other bit changes."""
    width, late = heads[2], min(rows, 2)
    p = Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths)
    clean, clean_weights = p.run(device, queue)
    values, prefix_values = p.v, p.pv
    for feature in (0, width // 2 + 3, width - 1):
        others = np.arange(width) != feature
        p.v = values.copy()
        for b, n in enumerate(lengths):  # seen by the last `late` rows
            p.v[b, n - late] = special_feature(oracle, dtype, values[b, n - late], feature, special)
        got, weights = p.run(device, queue)
        assert same_bits(got[..., others], clean[..., others])
        assert same_bits(got[:, :rows - late], clean[:, :rows - late])
        assert np.array_equal(value_of(got[:, rows - late:, :, feature]),
                              np.full((batch, late, heads[0]), special), equal_nan=True)
        assert same_bits(weights, clean_weights)
        p.v, p.pv = values, prefix_values.copy()
        if not prefix:
            continue
        p.pv[prefix - 2] = special_feature(oracle, dtype, p.pv[prefix - 2], feature, special)
        got, weights = p.run(device, queue)
        assert same_bits(got[..., others], clean[..., others])
        assert np.array_equal(value_of(got[..., feature]), np.full((batch, rows, heads[0]), special), equal_nan=True)
        assert same_bits(weights, clean_weights)
        p.pv = prefix_values


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


@types
@pytest.mark.parametrize("batch,rows,prefix,capacity,heads,lengths", [
    (9, 1, 1000, 4096, (8, 2, 128), [5, 4, 3, 2, 1, 0, 5, 300, 5]),
    (2, 1, 3000, 20000, (8, 2, 64), [200, 31]),
    (2, 20, 700, 9000, (8, 2, 128), [150, 40]),
    (1, 66, 8100, 5000, (8, 8, 128), [69]),
    (3, 16, 1001, 8192, (8, 2, 128), [115, 16, 40]),
    (1, 1, 0, 1 << 20, (2, 1, 8), [129]),
])
def test_caches_with_room_left(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths):
    """Caches of many more slots than rows in use, as a program allocates them: ranges and the join go by the slots."""
    Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths).check(device, queue)


@types
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("apart", range(6))
def test_attention_with_one_operand_off_alignment(device, queue, oracle, dtype, rows, apart):
    """An element past an aligned address for one of the query, the prefix, the cache and the output."""
    p = Problem(oracle, dtype, 2, rows, 40, 90, (8, 2, 128), [90, 41])
    out, bound, _, _ = p.want()
    at = [up(device, queue, x, int(i == apart)) for i, x in enumerate((p.q, p.pk, p.pv, p.k, p.v, np.zeros_like(p.q)))]
    lengths, scale = up(device, queue, p.lengths), up(device, queue, np.array([p.scale]))
    room = workspace_bytes("dl_attention_shared", p.shape, p.prefix)
    work = device.allocate(room)
    _lib.call("dl_attention_shared", queue.handle, CODE[dtype], C.byref(p.shape), *[x[1] for x in at[:3]], p.prefix, at[3][1],
              at[4][1], lengths[1], at[5][1], scale[1], work.ptr(), room)
    raw = queue.read(at[5][0], p.q.dtype, p.q.size + int(apart == 5) + 1)
    assert raw[-1] == 0 and (apart < 5 or raw[0] == 0)  # what lies beside the output stays
    got = raw[int(apart == 5):-1].reshape(p.q.shape)
    assert np.all(np.abs(value_of(got) - out) <= bound)


@types
@pytest.mark.parametrize("width", [64, 128, 12])
@pytest.mark.parametrize("apart", ["q", "k", "v", "q2", "keys", "values"])
def test_append_with_one_operand_off_alignment(device, queue, oracle, dtype, width, apart):
    """The bits of the aligned call, whichever operand lies an element past an aligned address."""
    batch, rows, capacity, qh, kvh = 2, 3, 11, 6, 2
    rng = np.random.default_rng(width)
    make = lambda *s: stored(oracle, rng.standard_normal(s), dtype)  # noqa: E731
    a = dict(q=make(batch, rows, qh, width), k=make(batch, rows, kvh, width), v=make(batch, rows, kvh, width))
    a.update(q2=np.zeros_like(a["q"]), keys=make(batch, capacity, kvh, width), values=make(batch, capacity, kvh, width),
             lengths=np.array([3, 9], np.uint64), lengths2=np.zeros(2, np.uint64), positions=np.array([70, 9], np.uint64),
             positions2=np.zeros(2, np.uint64), slots=np.zeros((batch, kvh, capacity), np.uint32),
             weights=np.ones((batch, kvh, capacity), np.float32))

    def run(off):
        b = {n: up(device, queue, x, int(n == off)) for n, x in a.items()}
        shape = BatchShape(batch, rows, qh, kvh, width, capacity)
        _lib.call("dl_cache_append", queue.handle, CODE[dtype], C.byref(shape), *[x[1] for x in b.values()], 1e6)
        whole = {n: queue.read(b[n][0], x.dtype, x.size + int(n == off) + 1) for n, x in a.items()}
        for n, x in whole.items():  # what lies beside an operand stays
            assert x[-1] == 0 and (n != off or x[0] == 0)
        return {n: x[int(n == off):-1] for n, x in whole.items()}

    want, got = run(None), run(apart)
    assert not np.array_equal(want["keys"], a["keys"].reshape(-1)) and np.any(want["q2"])
    for n in a:
        assert same_bits(got[n], want[n]), n


@types
@pytest.mark.parametrize("width", [128, 12])
@pytest.mark.parametrize("apart", ["keys", "values"])
def test_evict_with_one_operand_off_alignment(device, queue, oracle, dtype, width, apart):
    batch, capacity, kvh, budget = 2, 90, 2, 41
    k, v, weights, slots = evict_inputs(oracle, dtype, batch, kvh, width, capacity, width)
    lengths = np.array([90, 60], np.uint64)
    shape = BatchShape(batch, 1, kvh, kvh, width, capacity)
    b = [up(device, queue, x, int(n == apart)) for n, x in (("keys", k), ("values", v))]
    n, w, at = (up(device, queue, x) for x in (lengths, weights, slots))
    room = workspace_bytes("dl_cache_evict", shape, budget)
    work = device.allocate(room)
    _lib.call("dl_cache_evict", queue.handle, CODE[dtype], C.byref(shape), b[0][1], b[1][1], n[1], n[1], at[1], at[1], w[1], w[1],
              budget, 2, 9, work.ptr(), room)
    want = want_evict(k, v, weights, slots, lengths, budget, 2, 9, True)
    for name, buf, e in zip(("keys", "values"), b, want):
        off = int(name == apart)
        raw = queue.read(buf[0], e.dtype, e.size + off + 1)
        assert raw[-1] == 0 and (not off or raw[0] == 0)
        assert same_bits(raw[off:-1], e.reshape(-1)), name
    for buf, e in zip((w, at, n), want[2:]):
        assert same_bits(queue.read(buf[0], e.dtype, e.size), e.reshape(-1))


# ------------------------------------------------------------ the cache object
@pytest.mark.parametrize("first", [0, 3])
def test_sinks_are_positions_of_the_sequence(device, queue, oracle, first):
    """`sinks` counts positions from the sequence's start: rows behind a prefix that holds them all are not sinks."""
    rows, budget, width = 10, 8, 8
    for sinks in (first, first + 2):
        cache = BatchCache(device, queue, 1, rows, 1, 1, width, first_position=first)
        q, k, v = (device.upload_array(queue, np.zeros(rows * width, np.uint16)) for _ in range(3))
        cache.append(q, k, v, q, rows)
        queue.write(cache.weights, np.arange(rows, dtype=np.float32))  # the first rows received least
        cache.evict(budget, sinks)
        slots = queue.read(cache.slots, np.uint32, rows)[:budget]
        gone = {first, first + 1} if sinks == first else {first + 2, first + 3}
        assert set(slots.tolist()) == set(range(first, first + rows)) - gone
        assert cache.used == [budget]


def test_used_counts_a_recorded_step_once(device, queue, oracle):
    """A step recorded through the object counts as one replay; the program adds the rows of the others."""
    batch, capacity, prefix, qh, kvh, w, replays = 2, 9, 20, 4, 2, 64, 4
    rng = np.random.default_rng(8)
    make = lambda *s: up(device, queue, stored(oracle, rng.standard_normal(s), "bf16"))[0]  # noqa: E731
    cache = BatchCache(device, queue, batch, capacity, qh, kvh, w, first_position=prefix)
    cache.set_prefix(make(prefix, kvh, w), make(prefix, kvh, w), prefix)
    q, k, v = make(batch, 1, qh, w), make(batch, 1, kvh, w), make(batch, 1, kvh, w)
    turned, out = device.allocate(batch * qh * w * 2), device.allocate(batch * qh * w * 2)

    def step():
        cache.append(q, k, v, turned)
        cache.attend(turned, out)

    step()  # allocates the workspace
    ids = device.upload_array(queue, np.arange(replays, dtype=np.uint32))
    token = device.allocate(4)
    handle = C.c_void_p()
    _lib.call("dl_sequence_create", queue.handle, replays, 0, 1, 1, C.byref(handle))
    try:
        _lib.call("dl_sequence_begin", handle, None, None, token.ptr(), 4, ids.ptr(), replays * 4, None, None, None, None)
        for stage in range(4):
            _lib.call("dl_sequence_begin_stage", handle, stage)
            if stage == 0:
                step()
            if stage == 3:
                _lib.call("dl_sequence_begin_selection", handle)
            _lib.call("dl_sequence_end_stage", handle)
        _lib.call("dl_sequence_complete", handle)
        _lib.call("dl_sequence_start", handle)
        _lib.call("dl_sequence_drain", handle)
    finally:
        _lib.call("dl_sequence_destroy", handle)
    cache.used = [n + replays - 1 for n in cache.used]
    assert cache.used == [int(n) for n in queue.read(cache.lengths, np.uint64, batch)] == [1 + replays] * batch
    assert list(queue.read(cache.positions, np.uint64, batch)) == [prefix + 1 + replays] * batch
