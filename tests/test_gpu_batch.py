"""The batch operations on the GPU against their formulas in 64 bits
(batch_reference.py): attention over a shared prefix and own caches, the
weight every cached row received, append and eviction."""
import ctypes as C

import numpy as np
import pytest

import batch_reference as ref
from dolittle_amd import _lib
from dolittle_amd.batch import BatchCache, BatchShape, workspace_bytes

pytestmark = pytest.mark.gpu
CODE = {"bf16": 1, "f32": 2}


def stored(oracle, x, dtype):
    x = np.asarray(x, np.float32)
    return oracle.bf16_from_f32(x) if dtype == "bf16" else x


def value_of(x):
    return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if x.dtype == np.uint16 else x.astype(np.float64)


def up(device, queue, array, shift=0):
    """The array on the device, `shift` elements past an aligned address."""
    flat = np.ascontiguousarray(array).reshape(-1)
    buf = device.upload_array(queue, np.concatenate([np.zeros(shift, flat.dtype), flat, np.zeros(1, flat.dtype)]))
    return buf, buf.ptr(shift * flat.itemsize)


class Problem:
    """Operands of one attention call; rows past a length are NaN, the output
    and the workspace start as garbage."""

    def __init__(self, oracle, dtype, batch, rows, prefix, capacity, heads, lengths, seed=0, spread=1.0):
        rng = np.random.default_rng(seed * 1009 + batch * 31 + rows * 7 + prefix + capacity)
        qh, kvh, w = heads
        self.dtype, self.lengths, self.prefix, self.oracle = dtype, np.array(lengths, np.uint64), prefix, oracle
        self.shape = BatchShape(batch, rows, qh, kvh, w, capacity)
        make = lambda *s: stored(oracle, rng.standard_normal(s) * spread, dtype)  # noqa: E731
        self.q = make(batch, rows, qh, w)
        self.pk, self.pv = make(prefix, kvh, w), make(prefix, kvh, w)
        self.k, self.v = make(batch, capacity, kvh, w), make(batch, capacity, kvh, w)
        nan = np.uint16(0x7fc0) if dtype == "bf16" else np.float32(np.nan)
        for b in range(batch):
            n = min(int(self.lengths[b]), capacity)
            self.k[b, n:], self.v[b, n:] = nan, nan
        self.scale = np.float32(1.0 / np.sqrt(w))
        self.weights = rng.random((batch, kvh, capacity)).astype(np.float32)

    def run(self, device, queue, weighted=True, shift=0, in_place=False):
        size = 2 if self.dtype == "bf16" else 4
        held = [up(device, queue, a, shift) for a in (self.q, self.pk, self.pv, self.k, self.v)]
        (_, q), (_, pk), (_, pv), (_, k), (_, v) = held
        lengths, scale = up(device, queue, self.lengths), up(device, queue, np.array([self.scale]))
        out = device.upload_array(queue, np.full((self.q.size + 8 + shift) * size, 0xAB, np.uint8))
        name = "dl_attention_weighted" if weighted else "dl_attention_shared"
        room = workspace_bytes(name, self.shape, self.prefix)
        work = device.upload_array(queue, np.full(room + 64, 0xFF, np.uint8))
        extra = ()
        if weighted:
            weights = up(device, queue, self.weights)
            weights_out = weights if in_place else up(device, queue, np.full(self.weights.shape, -7.0, np.float32))
            extra = weights[1], weights_out[1]
        if not self.prefix:
            pk = pv = None
        _lib.call(name, queue.handle, CODE[self.dtype], C.byref(self.shape), q, pk, pv, self.prefix, k, v, lengths[1], *extra,
                  out.ptr(shift * size), scale[1], work.ptr(), room)
        queue.drain()
        raw = queue.read(out, np.uint8, out.nbytes)
        assert np.all(raw[:shift * size] == 0xAB) and np.all(raw[(shift + self.q.size) * size:] == 0xAB)
        assert np.all(queue.read(work, np.uint8, 64, room) == 0xFF)
        got = raw[shift * size:(shift + self.q.size) * size].view(self.q.dtype).reshape(self.q.shape)
        if not weighted:
            return got, None
        return got, queue.read(weights_out[0], np.float32, self.weights.size).reshape(self.weights.shape)

    def want(self):
        return ref.attention(*(value_of(x) for x in (self.q, self.pk, self.pv, self.k, self.v)), self.lengths,
                             float(self.scale), self.dtype)

    def check(self, device, queue, **how):
        out, bound, received, received_bound = self.want()
        got, weights = self.run(device, queue, **how)
        off = np.abs(value_of(got) - out)
        assert np.all(off <= bound), (float(np.max(off / bound)), np.argwhere(off > bound)[:4])
        if weights is not None:
            used = np.arange(weights.shape[2]) < np.minimum(self.lengths, weights.shape[2])[:, None, None].astype(np.int64)
            used = np.broadcast_to(used, weights.shape)
            total = self.weights + received
            wide = received_bound + 2.0 ** -23 * np.abs(total)
            off = np.abs(weights - total)[used]
            assert np.all(off <= wide[used]), float(np.max(off / wide[used]))
            kept = self.weights if how.get("in_place") else np.full(weights.shape, -7.0, np.float32)
            assert np.array_equal(weights[~used], kept[~used])


SHAPES = [
    # batch, rows, prefix, capacity, (query heads, KV heads, width), lengths
    (1, 1, 0, 1, (1, 1, 128), [1]),
    (1, 1, 0, 1, (1, 1, 128), [0]),  # no key at all
    (1, 1, 1, 4, (4, 4, 64), [0]),
    (2, 1, 31, 40, (8, 2, 128), [7, 0]),
    (3, 1, 33, 129, (12, 4, 128), [129, 128, 1]),
    (8, 1, 192, 24, (32, 8, 128), [24, 16, 21, 7, 24, 13, 19, 1]),
    (5, 1, 127, 300, (10, 2, 128), [300, 257, 1 << 40, 31, 32]),  # a length above the capacity
    (9, 1, 1000, 5, (8, 2, 128), [5, 4, 3, 2, 1, 0, 5, 5, 5]),
    (17, 1, 513, 8, (8, 2, 64), list(range(9)) + [8] * 8),
    (2, 2, 0, 70, (4, 1, 128), [70, 1]),  # fewer rows held than new ones: the first new row sees nothing
    (2, 5, 40, 70, (6, 2, 128), [5, 66]),
    (1, 16, 1001, 115, (32, 8, 128), [115]),
    (1, 67, 0, 201, (8, 2, 128), [201]),
    (3, 33, 5, 160, (4, 2, 64), [33, 160, 2]),
    (1, 1, 2049, 1, (16, 1, 256), [1]),
    (2, 9, 65, 90, (8, 1, 256), [90, 9]),
    (2, 1, 66, 35, (4, 2, 96), [35, 3]),
    (2, 20, 66, 135, (10, 2, 80), [135, 30]),
    (2, 3, 10, 40, (6, 3, 8), [40, 3]),
    (1, 2, 10, 40, (2, 1, 200), [40]),
    (2, 2, 17, 37, (4, 2, 1), [37, 2]),
    (2, 3, 17, 37, (4, 2, 20), [37, 2]),
    (1, 18, 17, 37, (4, 2, 65), [37]),
    (1, 2, 33, 37, (3, 1, 255), [36]),
    # Many rows, in BF16 64 or 128 a workgroup that shares its keys: prefix and
    # own cache, both forms on one or the other, each width and piece count.
    (1, 65, 0, 160, (4, 1, 128), [160]),
    (70, 1, 300, 40, (4, 2, 128), [40 - b % 41 for b in range(70)]),
    (40, 1, 129, 33, (6, 3, 96), [33 - b % 34 for b in range(40)]),
    (9, 1, 700, 33, (8, 1, 256), [33, 0, 1, 2, 3, 32, 31, 30, 5]),
    (5, 17, 100, 97, (3, 1, 248), [97, 17, 5, 96, 64]),
    (1, 129, 1024, 320, (8, 8, 64), [320]),
    (1, 140, 8200, 141, (8, 8, 64), [141]),
    (3, 33, 8100, 40, (16, 8, 128), [40, 33, 1]),
    (35, 1, 8192, 9, (16, 8, 88), [9 - b % 10 for b in range(35)]),
    (2, 80, 0, 2100, (16, 8, 40), [2100, 81]),
    (1, 150, 0, 4200, (16, 8, 128), [4133]),
    (17, 1, 8192, 3, (32, 8, 128), [3 - b % 4 for b in range(17)]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,rows,prefix,capacity,heads,lengths", SHAPES)
def test_attention(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths):
    p = Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths)
    p.check(device, queue)
    p.check(device, queue, in_place=True)
    got, _ = p.run(device, queue, weighted=True)
    alone, _ = p.run(device, queue, weighted=False)
    assert np.array_equal(got.view(np.uint8), alone.view(np.uint8))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,rows,prefix,capacity,heads,lengths",
                         [(3, 1, 33, 129, (12, 4, 128), [129, 128, 1]), (2, 9, 65, 90, (8, 1, 64), [90, 9])])
def test_operands_off_alignment(device, queue, oracle, dtype, batch, rows, prefix, capacity, heads, lengths):
    Problem(oracle, dtype, batch, rows, prefix, capacity, heads, lengths).check(device, queue, shift=1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_wide_scores(device, queue, oracle, dtype):
    """Scores of some hundreds: the running maximum rises often, and most weights underflow."""
    Problem(oracle, dtype, 2, 3, 700, 300, (8, 2, 128), [300, 150], spread=5.0).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(4, 1, 128), (2, 2, 20)])
def test_unseen_keys_leave_no_trace(device, queue, oracle, dtype, heads):
    """Infinities and NaN in the keys and values of the last new rows reach the
    rows that see them and no others."""
    rows, n = 6, 45
    p = Problem(oracle, dtype, 2, rows, 10, 50, heads, [n, n])
    clean, _ = p.run(device, queue, weighted=False)
    for special in (np.inf, -np.inf, np.nan):
        for operand in ("k", "v"):
            q = Problem(oracle, dtype, 2, rows, 10, 50, heads, [n, n])
            getattr(q, operand)[:, n - 2] = stored(oracle, np.full(heads[2], special), dtype)
            got, _ = q.run(device, queue, weighted=False)
            assert np.array_equal(got[:, :rows - 2].view(np.uint8), clean[:, :rows - 2].view(np.uint8))
            last = value_of(got[:, rows - 2:])
            if operand == "v":
                want = np.full_like(last, special)
                assert np.array_equal(last, want, equal_nan=True)
            elif np.isnan(special):
                assert np.all(np.isnan(last))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_special_scores(device, queue, oracle, dtype):
    """Visible keys whose scores are all -inf, one +inf or NaN give NaN, as the
    formula does; one -inf among finite ones has no weight."""
    p = Problem(oracle, dtype, 4, 1, 0, 40, (2, 1, 64), [40] * 4)
    p.q[:] = stored(oracle, np.ones(p.q.shape), dtype)
    inf = lambda v: stored(oracle, np.full(64, v), dtype)  # noqa: E731
    p.k[0, :], p.k[1, 3], p.k[2, 39], p.k[3, 17] = inf(-np.inf), inf(np.inf), inf(np.nan), inf(-np.inf)
    got, weights = p.run(device, queue)
    assert np.all(np.isnan(value_of(got[:3])))
    left = Problem(oracle, dtype, 1, 1, 0, 39, (2, 1, 64), [39])
    left.q, left.scale = p.q[3:], p.scale
    keep = [j for j in range(40) if j != 17]
    left.k, left.v = p.k[3:, keep], p.v[3:, keep]
    out, bound, _, _ = left.want()
    assert np.all(np.abs(value_of(got[3:]) - out) <= bound)
    assert weights[3, 0, 17] == p.weights[3, 0, 17]


def test_same_call_gives_the_same_bits(device, queue, oracle):
    p = Problem(oracle, "bf16", 8, 1, 1500, 700, (32, 8, 128), [700, 1, 350, 699, 128, 129, 512, 0])
    first, second = p.run(device, queue), p.run(device, queue)
    assert np.array_equal(first[0], second[0]) and np.array_equal(first[1], second[1])


def test_two_queues_at_once(device, queue, oracle):
    other = device.create_queue()
    p = Problem(oracle, "bf16", 4, 1, 3000, 500, (32, 8, 128), [500, 2, 77, 400])
    want, _ = p.run(device, queue, weighted=False)
    size = workspace_bytes("dl_attention_shared", p.shape, p.prefix)
    common = [up(device, queue, a)[0] for a in (p.q, p.pk, p.pv, p.k, p.v)]
    lengths, scale = up(device, queue, p.lengths)[0], up(device, queue, np.array([p.scale]))[0]
    outs = [device.allocate(p.q.nbytes) for _ in range(2)]
    works = [device.allocate(size) for _ in range(2)]
    for _ in range(20):
        for on, out, work in zip((queue, other), outs, works):
            q, pk, pv, k, v = (b.ptr() for b in common)
            _lib.call("dl_attention_shared", on.handle, 1, C.byref(p.shape), q, pk, pv, p.prefix, k, v, lengths.ptr(),
                      out.ptr(), scale.ptr(), work.ptr(), size)
    queue.drain()
    other.drain()
    for out in outs:
        assert np.array_equal(queue.read(out, np.uint16, p.q.size).reshape(p.q.shape), want)


def zeros(device, queue, nbytes):
    buf = device.allocate(nbytes)
    done = min(nbytes, 1 << 24)
    queue.write(buf, np.zeros(done, np.uint8))
    while done < nbytes:
        more = min(done, nbytes - done)
        queue.copy(buf, buf, more, done, 0)
        done += more
    return buf


def test_caches_past_32_bit_offsets(device, queue, oracle):
    """The second sequence's rows lie past 2^32 bytes, and past 2^31 elements."""
    heads, width, capacity, n = 8, 128, 2_200_000, 2_100_000
    row = heads * width * 2
    k, v = (zeros(device, queue, 2 * capacity * row) for _ in range(2))
    put = lambda buf, at, x: queue.write(buf, stored(oracle, np.full(heads * width, x), "bf16"), (capacity + at) * row)  # noqa: E731
    put(v, 17, 1.0)
    put(v, n - 1, 3.0)
    put(v, n, np.nan)
    put(k, n - 1, 0.5)
    q = device.upload_array(queue, stored(oracle, np.full(2 * heads * width, 0.5), "bf16"))
    out, scale = device.allocate(2 * row), device.upload_array(queue, np.ones(1, np.float32))
    lengths = device.upload_array(queue, np.array([1, n], np.uint64))
    weights = zeros(device, queue, 2 * heads * capacity * 4)
    shape = BatchShape(2, 1, heads, heads, width, capacity)
    size = workspace_bytes("dl_attention_weighted", shape, 0)
    work = device.allocate(size)
    _lib.call("dl_attention_weighted", queue.handle, 1, C.byref(shape), q.ptr(), None, None, 0, k.ptr(), v.ptr(),
              lengths.ptr(), weights.ptr(), weights.ptr(), out.ptr(), scale.ptr(), work.ptr(), size)
    queue.drain()
    # One score of 32, the others 0.  Sums of FP32 ones are exact here; the largest weight and the
    # sum over the joined ranges carry a few steps.
    e = np.exp(32.0)
    total = e + n - 1
    got = value_of(queue.read(out, np.uint16, 2 * heads * width)).reshape(2, -1)
    assert np.all(np.abs(got[1] - (3.0 * e + 1.0) / total) <= 2 * 2.0 ** -8 * 3.0) and np.all(got[0] == 0.0)
    got = queue.read(weights, np.float32, 2 * heads * capacity).reshape(2, heads, capacity)[1].astype(np.float64)
    assert np.all(np.abs(got[:, n - 1] - e / total) <= 1e-5)
    assert np.all(np.abs(got[:, [0, 17, n - 2]] * total - 1.0) <= 1e-4) and np.all(got[:, n:] == 0.0)


# ------------------------------------------------------------------- eviction
def evict_inputs(oracle, dtype, batch, kv_heads, width, capacity, seed):
    rng = np.random.default_rng(seed)
    rows = (batch, capacity, kv_heads, width)
    k, v = (stored(oracle, rng.standard_normal(rows), dtype) for _ in range(2))
    weights = (rng.integers(0, 40, (batch, kv_heads, capacity)) / 8).astype(np.float32)
    slots = np.stack([np.stack([rng.permutation(2 * capacity)[:capacity] for _ in range(kv_heads)])
                      for _ in range(batch)]).astype(np.uint32)
    return k, v, weights, slots


def run_evict(device, queue, dtype, k, v, weights, slots, lengths, budget, sinks, recent, in_place, shift=0):
    batch, capacity, kv_heads, width = k.shape
    shape = BatchShape(batch, 1, kv_heads, kv_heads, width, capacity)
    bk, bv = up(device, queue, k, shift), up(device, queue, v, shift)
    n, w, s = up(device, queue, lengths), up(device, queue, weights), up(device, queue, slots)
    fill = lambda x, value: up(device, queue, np.full(x.shape, value, x.dtype))  # noqa: E731
    n2, w2, s2 = (n, w, s) if in_place else (fill(lengths, 99), fill(weights, -7.0), fill(slots, 12345))
    room = workspace_bytes("dl_cache_evict", shape, budget)
    work = device.upload_array(queue, np.full(room + 64, 0xFF, np.uint8))
    _lib.call("dl_cache_evict", queue.handle, CODE[dtype], C.byref(shape), bk[1], bv[1], n[1], n2[1], s[1], s2[1], w[1], w2[1],
              budget, sinks, recent, work.ptr(), room)
    queue.drain()
    assert np.all(queue.read(work, np.uint8, 64, room) == 0xFF)
    read = lambda b, like, at=0: queue.read(b[0], like.dtype, like.size, at * like.itemsize).reshape(like.shape)  # noqa: E731
    return read(bk, k, shift), read(bv, v, shift), read(w2, weights), read(s2, slots), read(n2, lengths)


def want_evict(k, v, weights, slots, lengths, budget, sinks, recent, in_place):
    k, v = k.copy(), v.copy()
    w2 = weights.copy() if in_place else np.full_like(weights, -7.0)
    s2 = slots.copy() if in_place else np.full_like(slots, 12345)
    left = []
    for b in range(k.shape[0]):
        n = min(int(lengths[b]), k.shape[1])
        left.append(min(n, budget))
        for h in range(k.shape[2]):
            source = ref.evict(weights[b, h], slots[b, h], n, budget, sinks, recent)
            m = len(source)
            k[b, :m, h], v[b, :m, h] = k[b, source, h], v[b, source, h]
            w2[b, h, :m], s2[b, h, :m] = weights[b, h, source], slots[b, h, source]
    return k, v, w2, s2, np.array(left, np.uint64)


EVICTIONS = [
    # batch, KV heads, width, capacity, lengths, budget, sinks, recent
    (1, 1, 8, 2, [2], 1, 0, 0),
    (1, 1, 8, 2, [2], 1, 0, 1),
    (2, 2, 16, 40, [40, 13], 17, 2, 5),
    (3, 4, 128, 130, [130, 100, 64], 64, 4, 60),  # all that stays is protected
    (2, 2, 64, 1100, [1025, 1024], 1000, 0, 0),
    (2, 1, 20, 3000, [2500, 3000], 2049, 1, 100),  # one round lies on both sides of the budget
    (4, 2, 8, 70, [0, 1, 70, 1 << 33], 69, 3, 3),
    (1, 2, 1, 33, [33], 5, 1, 1),
    (1, 2, 8, 50, [50], 60, 1, 1),  # a budget above the capacity
    (1, 2, 8, 50, [50], (1 << 64) - 1, 1, (1 << 64) - 3),
    (1, 1, 8, 70000, [69999], 1500, 10, 40),
    (1, 1, 8, 70000, [70000], 69001, 10, 40),
    (1, 2, 8, 36864, [36864], 20000, 0, 1),  # the longest cache whose keys are held on chip
    (1, 2, 8, 36865, [36865], 20000, 0, 1),
    (1, 2, 8, 1024, [1024], 512, 0, 1),
    (1, 2, 8, 1025, [1025], 1024, 0, 1),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,kv_heads,width,capacity,lengths,budget,sinks,recent", EVICTIONS)
def test_evict(device, queue, oracle, dtype, in_place, batch, kv_heads, width, capacity, lengths, budget, sinks, recent):
    lengths = np.array(lengths, np.uint64)
    k, v, w, s = evict_inputs(oracle, dtype, batch, kv_heads, width, capacity, capacity + budget % 1000)
    for shift in (0, 1):
        got = run_evict(device, queue, dtype, k, v, w, s, lengths, budget, sinks, recent, in_place, shift)
        want = want_evict(k, v, w, s, lengths, budget, sinks, recent, in_place)
        for name, g, e in zip(("keys", "values", "weights", "slots", "lengths"), got, want):
            assert np.array_equal(g.view(np.uint8), e.view(np.uint8)), name


@pytest.mark.parametrize("kind", ["equal", "special", "protected_nan", "negative"])
def test_evict_orders(device, queue, oracle, kind):
    """Equal weights go by slot; NaN orders as -infinity, the zeros alike; a
    protected row stays whatever its weight."""
    k, v, w, s = evict_inputs(oracle, "bf16", 1, 2, 16, 600, 5)
    rng = np.random.default_rng(9)
    if kind == "equal":
        w[:] = 1.5
    elif kind == "special":
        w[:] = rng.choice(np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, 3e38], np.float32), w.shape)
    elif kind == "protected_nan":
        w[:] = np.where(s < 40, np.float32(np.nan), w)
    else:
        w[:] = rng.standard_normal(w.shape) * np.exp(rng.standard_normal(w.shape) * 20)
    lengths = np.array([600], np.uint64)
    for budget in (1, 299, 300, 599):
        sinks, recent = min(40, budget // 2), min(30, budget // 3)
        got = run_evict(device, queue, "bf16", k, v, w, s, lengths, budget, sinks, recent, False)
        want = want_evict(k, v, w, s, lengths, budget, sinks, recent, False)
        for name, g, e in zip(("keys", "values", "weights", "slots", "lengths"), got, want):
            assert np.array_equal(g.view(np.uint8), e.view(np.uint8)), (name, budget)


def test_evict_signalling_nan_weights(device, queue, oracle):
    """Every NaN orders as -infinity, whatever its bits."""
    k, v, w, s = evict_inputs(oracle, "bf16", 2, 1, 16, 500, 6)
    bits = np.array([0x7f800001, 0x7fbfffff, 0x7fffffff, 0xff800001, 0xffffffff, 0xffc00000], np.uint32)
    rng = np.random.default_rng(10)
    at = rng.random(w.shape) < 0.5
    w.view(np.uint32)[at] = rng.choice(bits, at.sum())
    lengths = np.array([500, 333], np.uint64)
    for budget in (100, 250, 480):
        got = run_evict(device, queue, "bf16", k, v, w, s, lengths, budget, 2, 9, False)
        want = want_evict(k, v, w, s, lengths, budget, 2, 9, False)
        for name, g, e in zip(("keys", "values", "weights", "slots", "lengths"), got, want):
            assert np.array_equal(g.view(np.uint8), e.view(np.uint8)), (name, budget)


@pytest.mark.parametrize("same", ["weights", "slots", "lengths"])
def test_evict_one_operand_in_place(device, queue, oracle, same):
    k, v, w, s = evict_inputs(oracle, "f32", 2, 2, 12, 90, 7)
    lengths, budget = np.array([90, 61], np.uint64), 50
    shape = BatchShape(2, 1, 2, 2, 12, 90)
    b = {n: up(device, queue, x) for n, x in dict(k=k, v=v, lengths=lengths, slots=s, weights=w).items()}
    for n, x in dict(lengths=lengths, slots=s, weights=w).items():
        b[n + "2"] = b[n] if n == same else up(device, queue, x)
    room = workspace_bytes("dl_cache_evict", shape, budget)
    work = device.allocate(room)
    order = ("k", "v", "lengths", "lengths2", "slots", "slots2", "weights", "weights2")
    _lib.call("dl_cache_evict", queue.handle, 2, C.byref(shape), *[b[n][1] for n in order], budget, 1, 5, work.ptr(), room)
    queue.drain()
    want = want_evict(k, v, w, s, lengths, budget, 1, 5, True)
    for n, e in zip(("k", "v", "weights2", "slots2", "lengths2"), want):
        assert np.array_equal(queue.read(b[n][0], e.dtype, e.size).reshape(e.shape).view(np.uint8), e.view(np.uint8)), n


# --------------------------------------------------------------------- append
APPENDS = [
    # batch, rows, capacity, (query heads, KV heads, width), lengths, positions
    (1, 1, 1, (1, 1, 2), [0], [0]),
    (8, 1, 40, (32, 8, 128), [0, 1, 39, 7, 8, 9, 30, 31], [0, 1, 4000, 32767, 8, 131071, 30, 31]),
    (2, 5, 16, (6, 2, 64), [3, 11], [3, 900]),
    (3, 7, 16, (4, 2, 80), [9, 10, 16], [9, 10, 5]),  # two sequences have no room for all
    (2, 3, 9, (4, 4, 6), [1 << 50, 2], [1, 2]),  # a length above the capacity
    (1, 70, 80, (3, 1, 256), [10], [1 << 20]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,rows,capacity,heads,lengths,positions", APPENDS)
def test_append(device, queue, oracle, dtype, in_place, batch, rows, capacity, heads, lengths, positions):
    """Rotated rows are dl_rotary's bits in FP32 storage, and those values
    rounded once in BF16; what no row enters stays."""
    qh, kvh, w = heads
    rng = np.random.default_rng(batch * 100 + rows)
    make = lambda *s: stored(oracle, rng.standard_normal(s), dtype)  # noqa: E731
    q, k, v = make(batch, rows, qh, w), make(batch, rows, kvh, w), make(batch, rows, kvh, w)
    keys, values = make(batch, capacity, kvh, w), make(batch, capacity, kvh, w)
    slots = rng.integers(0, 1 << 32, (batch, kvh, capacity), dtype=np.uint32)
    weights = rng.random((batch, kvh, capacity)).astype(np.float32)
    lengths, positions = np.array(lengths, np.uint64), np.array(positions, np.uint64)
    size = q.itemsize
    shape = BatchShape(batch, rows, qh, kvh, w, capacity)
    b = {n: up(device, queue, a) for n, a in dict(q=q, k=k, v=v, keys=keys, values=values, slots=slots, weights=weights,
                                                    lengths=lengths, positions=positions).items()}
    if in_place:
        b.update(q2=b["q"], lengths2=b["lengths"], positions2=b["positions"])
    else:
        b.update(q2=up(device, queue, np.zeros_like(q)), lengths2=up(device, queue, np.zeros_like(lengths)),
                 positions2=up(device, queue, np.zeros_like(positions)))
    want_q, want_k = np.empty_like(q), np.empty_like(k)
    for i in range(batch):  # one sequence at a time through the catalog's rotary
        for x, into, h in ((q, want_q, qh), (k, want_k, kvh)):
            wide = value_of(x[i]).astype(np.float32)
            src, dst = up(device, queue, wide), device.allocate(wide.nbytes)
            _lib.call("dl_rotary", queue.handle, 2, src[1], dst.ptr(), rows, h, w, int(positions[i]), 1e6, None, 0)
            into[i] = stored(oracle, queue.read(dst, np.float32, wide.size).reshape(wide.shape), dtype)
    order = ("q", "k", "v", "q2", "keys", "values", "lengths", "lengths2", "positions", "positions2", "slots", "weights")
    _lib.call("dl_cache_append", queue.handle, CODE[dtype], C.byref(shape), *[b[n][1] for n in order], 1e6)
    queue.drain()
    for i in range(batch):
        n = min(int(lengths[i]), capacity)
        for r in range(rows):
            if int(lengths[i]) + r < capacity:
                keys[i, n + r], values[i, n + r] = want_k[i, r], v[i, r]
                slots[i, :, n + r], weights[i, :, n + r] = int(positions[i]) + r, 0.0
    grown = np.array([min(min(int(n), capacity) + rows, capacity) for n in lengths], np.uint64)
    for n, e in (("q2", want_q), ("keys", keys), ("values", values), ("slots", slots), ("weights", weights),
                 ("lengths2", grown), ("positions2", positions + np.uint64(rows))):
        assert np.array_equal(queue.read(b[n][0], e.dtype, e.size).reshape(e.shape).view(np.uint8), e.view(np.uint8)), n


# ------------------------------------------------------------ used together
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_with_bounded_caches(device, queue, oracle, dtype):
    """Samples of one prompt with caches cut whenever they pass a budget:
    prompt chunk, decode steps, evictions, each step against the formulas over
    the rows that the host's own bookkeeping says are held."""
    batch, prefix, capacity, budget, sinks, recent = 3, 37, 24, 12, 2, 4
    qh, kvh, w = 8, 2, 64
    rng = np.random.default_rng(11)
    make = lambda *s: stored(oracle, rng.standard_normal(s), dtype)  # noqa: E731
    cache = BatchCache(device, queue, batch, capacity, qh, kvh, w, dtype, first_position=prefix)
    pk, pv = make(prefix, kvh, w), make(prefix, kvh, w)
    bpk, bpv = up(device, queue, pk)[0], up(device, queue, pv)[0]
    cache.set_prefix(bpk, bpv, prefix)
    scale = np.float32(1.0 / np.sqrt(np.float64(w)))
    totals = np.zeros((batch, kvh, capacity))
    for step, rows in enumerate([7, 1, 1, 3, 1, 1, 1, 5, 1, 1, 1, 1]):
        q, k, v = make(batch, rows, qh, w), make(batch, rows, kvh, w), make(batch, rows, kvh, w)
        held = [up(device, queue, x)[0] for x in (q, k, v)]
        turned, out = device.allocate(q.nbytes), device.allocate(q.nbytes)
        cache.append(*held, turned, rows)
        cache.attend(turned, out, rows)
        n = cache.used[0]
        read = lambda buf, t, s: queue.read(buf, t, int(np.prod(s))).reshape(s)  # noqa: E731
        tq = read(turned, q.dtype, q.shape)
        keys, values = (read(x, q.dtype, (batch, capacity, kvh, w)) for x in (cache.keys, cache.values))
        assert np.array_equal(values[:, n - rows:n], v)
        want, bound, received, wide = ref.attention(*(value_of(x) for x in (tq, pk, pv, keys, values)), [n] * batch,
                                                    float(scale), dtype)
        got = value_of(read(out, q.dtype, q.shape))
        assert np.all(np.abs(got - want) <= bound)
        totals[:, :, n - rows:n] = 0.0
        weights = read(cache.weights, np.float32, (batch, kvh, capacity))
        expect = totals + received
        assert np.all(np.abs(weights - expect)[:, :, :n] <= (wide + 2.0 ** -23 * expect)[:, :, :n])
        totals[:, :, :n] = weights[:, :, :n]
        slots = read(cache.slots, np.uint32, (batch, kvh, capacity))
        if n > budget:
            expected = want_evict(keys, values, weights, slots, [n] * batch, budget, sinks, recent, True)
            cache.evict(budget, sinks, recent)
            after = [read(cache.keys, q.dtype, keys.shape), read(cache.values, q.dtype, values.shape),
                     read(cache.weights, np.float32, weights.shape), read(cache.slots, np.uint32, slots.shape),
                     read(cache.lengths, np.uint64, (batch,))]
            for g, e in zip(after, expected):
                assert np.array_equal(g.view(np.uint8), e.view(np.uint8))
            totals[:, :, :budget] = after[2][:, :, :budget]
            newest = prefix + sum([7, 1, 1, 3, 1, 1, 1, 5, 1, 1, 1, 1][:step + 1]) - 1
            assert np.all(np.isin(np.arange(newest - recent + 1, newest + 1), after[3][0, 0, :budget]))
    assert cache.used == [int(x) for x in queue.read(cache.lengths, np.uint64, batch)]
    with pytest.raises(_lib.LengthError):
        cache.append(None, None, None, None, capacity)


def test_steps_replayed_from_graphs(device, queue, oracle):
    """Append, weighted attention and eviction recorded once into a sequence's
    graphs and replayed nine times, twice, with eager work between: the bits of
    the same steps submitted one by one."""
    batch, prefix, capacity, budget, heads, steps = 3, 70, 9, 8, (8, 2, 64), 9
    qh, kvh, w = heads
    rng = np.random.default_rng(3)
    make = lambda *s: stored(oracle, rng.standard_normal(s), "bf16")  # noqa: E731
    pk, pv = (up(device, queue, make(prefix, kvh, w))[0] for _ in range(2))
    q, k, v = (up(device, queue, make(batch, 1, h, w))[0] for h in (qh, kvh, kvh))
    start = make(batch, capacity, kvh, w), make(batch, capacity, kvh, w)

    class Side:
        def __init__(self):
            self.cache = BatchCache(device, queue, batch, capacity, qh, kvh, w, first_position=prefix)
            for buf, x in zip((self.cache.keys, self.cache.values), start):
                queue.write(buf, x)
            for buf in (self.cache.weights, self.cache.slots):
                queue.write(buf, np.zeros(batch * kvh * capacity, np.float32))
            self.turned, self.out = (device.allocate(batch * qh * w * 2) for _ in range(2))
            shape = self.cache.shape()
            rooms = [workspace_bytes("dl_attention_weighted", shape, prefix), workspace_bytes("dl_cache_evict", shape, budget)]
            self.work = [device.upload_array(queue, np.full(n, 0xFF, np.uint8)) for n in rooms]

        def step(self):
            c, shape = self.cache, self.cache.shape()
            _lib.call("dl_cache_append", queue.handle, 1, C.byref(shape), q.ptr(), k.ptr(), v.ptr(), self.turned.ptr(),
                      c.keys.ptr(), c.values.ptr(), c.lengths.ptr(), c.lengths.ptr(), c.positions.ptr(), c.positions.ptr(),
                      c.slots.ptr(), c.weights.ptr(), 1e6)
            _lib.call("dl_attention_weighted", queue.handle, 1, C.byref(shape), self.turned.ptr(), pk.ptr(), pv.ptr(), prefix,
                      c.keys.ptr(), c.values.ptr(), c.lengths.ptr(), c.weights.ptr(), c.weights.ptr(), self.out.ptr(),
                      c._scale.ptr(), self.work[0].ptr(), self.work[0].nbytes)
            _lib.call("dl_cache_evict", queue.handle, 1, C.byref(shape), c.keys.ptr(), c.values.ptr(), c.lengths.ptr(),
                      c.lengths.ptr(), c.slots.ptr(), c.slots.ptr(), c.weights.ptr(), c.weights.ptr(), budget, 1, 2,
                      self.work[1].ptr(), self.work[1].nbytes)

        def state(self):
            c = self.cache
            return [queue.read(b, np.uint8, b.nbytes) for b in (c.keys, c.values, c.weights, c.slots, c.lengths, c.positions,
                                                                self.out)]

    eager, replayed = Side(), Side()
    ids = device.upload_array(queue, np.arange(steps, dtype=np.uint32))
    token = device.allocate(4)
    for _ in range(2):
        handle = C.c_void_p()
        _lib.call("dl_sequence_create", queue.handle, steps, 0, 1, 1, C.byref(handle))
        try:
            _lib.call("dl_sequence_begin", handle, None, None, token.ptr(), 4, ids.ptr(), steps * 4, None, None, None, None)
            for stage in range(4):
                _lib.call("dl_sequence_begin_stage", handle, stage)
                if stage == 0:
                    replayed.step()
                if stage == 3:
                    _lib.call("dl_sequence_begin_selection", handle)
                _lib.call("dl_sequence_end_stage", handle)
            _lib.call("dl_sequence_complete", handle)
            _lib.call("dl_sequence_start", handle)
            _lib.call("dl_sequence_drain", handle)
        finally:
            _lib.call("dl_sequence_destroy", handle)
        for _ in range(steps):
            eager.step()
        queue.drain()
        for got, want in zip(replayed.state(), eager.state()):
            assert np.array_equal(got, want)
    assert list(queue.read(eager.cache.positions, np.uint64, batch)) == [prefix + 2 * steps] * batch


def test_cache_object_refusals(device, queue):
    from dolittle_amd import InvalidArgument, LengthError
    for bad in (dict(batch=0), dict(capacity=0), dict(width=0), dict(dtype="f16"), dict(first_position=-1)):
        with pytest.raises(InvalidArgument):
            BatchCache(device, queue, **{**dict(batch=1, capacity=4, query_heads=2, kv_heads=1, width=8), **bad})
    cache = BatchCache(device, queue, 1, 4, 2, 1, 8)
    x = device.allocate(256)
    with pytest.raises(LengthError):
        cache.append(x, x, x, x, 5)
    with pytest.raises(InvalidArgument):
        cache.append(x, x, x, x, 0)
    with pytest.raises(InvalidArgument):
        cache.append(None, x, x, x)
    assert cache.used == [0]
    for budget, sinks, recent in ((0, 0, 0), (3, 2, 2), (3, -1, 0)):
        with pytest.raises(InvalidArgument):
            cache.evict(budget, sinks, recent)
    with pytest.raises(InvalidArgument):
        cache.attend(None, x)
