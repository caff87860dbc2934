"""The operations over 4-bit storage on the GPU against their formulas in 64 bits
(fp4_reference.py): quantising and reading back, the projection, the append and
the attention with and without a window."""
import ctypes as C

import numpy as np
import pytest

import fp4_reference as ref
from dolittle_amd import LengthError, _lib
from dolittle_amd.batch import BatchShape
from dolittle_amd.fp4 import CacheAddresses, Fp4Cache, Fp4Weight, attention_workspace_bytes

pytestmark = pytest.mark.gpu
CODE = {"bf16": 1, "f32": 2}
SIZE = {"bf16": 2, "f32": 4}


def stored(oracle, x, dtype):
    x = np.asarray(x, np.float32)
    return oracle.bf16_from_f32(x) if dtype == "bf16" else x


def value_of(x):
    with np.errstate(invalid="ignore"):
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if x.dtype == np.uint16 else x.astype(np.float64)


def up(device, queue, array, shift=0):
    """The array on the device, `shift` elements past an aligned address."""
    flat = np.ascontiguousarray(array).reshape(-1)
    buf = device.upload_array(queue, np.concatenate([np.zeros(shift, flat.dtype), flat, np.zeros(1, flat.dtype)]))
    return buf, buf.ptr(shift * flat.itemsize)


class Room:
    """Device memory of some elements between guard bytes, for results."""

    def __init__(self, device, queue, count, dtype, shift=0):
        self.queue, self.count, self.dtype = queue, count, np.dtype(dtype)
        self.before, self.bytes = 64 + shift * self.dtype.itemsize, count * self.dtype.itemsize
        self.buffer = device.upload_array(queue, np.full(self.before + self.bytes + 64, 0xAB, np.uint8))
        self.at = self.buffer.ptr(self.before)

    def read(self):
        self.queue.drain()
        raw = self.queue.read(self.buffer, np.uint8, self.buffer.nbytes)
        assert np.all(raw[:self.before] == 0xAB) and np.all(raw[self.before + self.bytes:] == 0xAB), "written outside"
        return raw[self.before:self.before + self.bytes].view(self.dtype)


def storage(dtype):
    return np.uint16 if dtype == "bf16" else np.float32


def same(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.nan_to_num(got, nan=0.0), np.nan_to_num(want, nan=0.0))


def close(got, want, bound):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(got - want)
    fine = np.isnan(want) | (off <= bound)
    assert fine.all(), f"off by {np.nanmax(off / np.maximum(bound, 1e-300)):.3g} bounds at {np.argwhere(~fine)[:4].tolist()}"


def packed_random(rng, shape, spread=1.0):
    """Codes and scales of normal rows."""
    return ref.quantized((rng.standard_normal(shape) * spread).astype(np.float32).astype(np.float64))


# ------------------------------------------------------ quantise and read back
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,width,shift", [(1, 1, 0), (3, 32, 0), (5, 80, 0), (2, 31, 0), (33, 1000, 0), (4, 256, 1), (64, 4096, 0),
                                              (7, 64, 3)])
def test_quantize_and_values(oracle, device, queue, dtype, rows, width, shift):
    rng = np.random.default_rng(rows * 1000 + width)
    x = stored(oracle, rng.standard_normal((rows, width)) * np.exp(rng.uniform(-20, 20, (rows, 1))), dtype)
    groups = ref.groups_of(width)
    held, at = up(device, queue, x, shift)
    codes, scales = Room(device, queue, rows * groups * 16, np.uint8), Room(device, queue, rows * groups, np.uint8, shift)
    _lib.call("dl_fp4_quantize", queue.handle, CODE[dtype], at, codes.at, scales.at, rows, width)
    want_codes, want_scales = ref.quantized(value_of(x))
    assert np.array_equal(scales.read().reshape(rows, groups), want_scales)
    assert np.array_equal(codes.read().reshape(rows, groups, 16), want_codes)
    for out_type in ("bf16", "f32"):
        out = Room(device, queue, rows * width, storage(out_type), shift)
        _lib.call("dl_fp4_values", queue.handle, CODE[out_type], codes.at, scales.at, out.at, rows, width)
        same(value_of(out.read()).reshape(rows, width), ref.values(want_codes, want_scales, width))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_borders_and_special_values(oracle, device, queue, dtype):
    """Ties between codes, every scale byte that quantising gives, subnormal, huge, infinite and NaN values."""
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    base = np.concatenate((borders, -borders, [0.0, -0.0, 0.5, 1, 1.5, 2, 3, 4, 6.5, 6.9375, -6.5, 0.2490234375, 0.251953125, -1.5, -2, -6]))
    rows = [np.ldexp(base, s - 127) for s in range(0, 252)]
    rows += [np.where(base == 6.0, v, base) for v in (np.nan, np.inf, -np.inf)]
    rows += [np.full(32, 3.3e38), np.full(32, -1e-40), np.zeros(32), np.full(32, 2.0 ** -149), np.full(32, -0.0)]
    rng = np.random.default_rng(5)
    rows += list(rng.standard_normal((64, 32)) * np.exp(rng.uniform(-60, 60, (64, 1))))
    x = stored(oracle, np.array(rows, np.float32), dtype)
    held, at = up(device, queue, x)
    codes, scales = Room(device, queue, len(rows) * 16, np.uint8), Room(device, queue, len(rows), np.uint8)
    _lib.call("dl_fp4_quantize", queue.handle, CODE[dtype], at, codes.at, scales.at, len(rows), 32)
    want_codes, want_scales = ref.quantized(value_of(x))
    assert np.array_equal(scales.read()[:, None], want_scales)
    assert np.array_equal(codes.read().reshape(-1, 1, 16), want_codes)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_values_of_every_code_and_scale(device, queue, dtype):
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(16, 16), (16, 1)).reshape(-1, 1, 16)
    for scale in (0, 1, 2, 64, 127, 128, 200, 251, 252, 255):
        scales = np.full((len(codes), 1), scale, np.uint8)
        (hc, c), (hs, s) = up(device, queue, codes), up(device, queue, scales)
        out = Room(device, queue, len(codes) * 32, storage(dtype))
        _lib.call("dl_fp4_values", queue.handle, CODE[dtype], c, s, out.at, len(codes), 32)
        same(value_of(out.read()).reshape(-1, 32), ref.values(codes, scales, 32))


# ----------------------------------------------------------------- projection
def project(device, queue, dtype, x, codes, scales, rows, inputs, outputs, shift=0, position=None):
    (hx, xa), (hc, c), (hs, s) = up(device, queue, x, shift), up(device, queue, codes), up(device, queue, scales, shift)
    first = position or 0
    out = Room(device, queue, (first + rows) * outputs, storage(dtype), shift)
    place = None if position is None else up(device, queue, np.array([position], np.uint64))
    _lib.call("dl_projection_fp4", queue.handle, CODE[dtype], xa, c, s, out.at, rows, inputs, outputs, place and place[1])
    got = out.read().reshape(first + rows, outputs)
    assert np.all(np.ascontiguousarray(got[:first]).view(np.uint8) == 0xAB)
    return value_of(got[first:])


PROJECTIONS = [(1, 32, 16), (1, 4096, 1024), (2, 1000, 777), (3, 12288, 33), (5, 31, 1), (8, 256, 4096), (16, 288, 50), (17, 4096, 64),
               (33, 160, 100), (64, 512, 129), (100, 2048, 300), (257, 96, 260), (130, 33, 65),
               (2, 8100, 40), (4, 6145, 20), (3, 12500, 37), (1, 30000, 16), (6, 1999, 2100), (1, 64, 9000)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,inputs,outputs", PROJECTIONS)
def test_projection(oracle, device, queue, dtype, rows, inputs, outputs):
    rng = np.random.default_rng(rows * 7 + inputs + outputs)
    x = stored(oracle, rng.standard_normal((rows, inputs)), dtype)
    codes, scales = packed_random(rng, (outputs, inputs), inputs ** -0.5)
    want, bound = ref.projection(value_of(x), ref.values(codes, scales, inputs), dtype)
    close(project(device, queue, dtype, x, codes, scales, rows, inputs, outputs), want, bound)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,position", [(1, 3), (20, 2)])
def test_projection_off_alignment_at_a_position(oracle, device, queue, dtype, rows, position):
    rng = np.random.default_rng(rows)
    x = stored(oracle, rng.standard_normal((rows, 320)), dtype)
    codes, scales = packed_random(rng, (48, 320))
    want, bound = ref.projection(value_of(x), ref.values(codes, scales, 320), dtype)
    close(project(device, queue, dtype, x, codes, scales, rows, 320, 48, 1, position), want, bound)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [3, 40])
def test_projection_special_values(oracle, device, queue, dtype, rows):
    """A NaN group reaches its output alone, a NaN or infinite input its row alone; scales far apart; garbage codes
    and whole-group NaN behind the last group are not there to be read."""
    rng = np.random.default_rng(11)
    codes, scales = packed_random(rng, (70, 320))
    scales[5, 7], scales[69, 0] = 255, 255
    scales[8] = rng.integers(40, 200, scales[8].shape)
    x = rng.standard_normal((rows, 320))
    x[1, 300], x[2, 4] = np.nan, np.inf
    x = stored(oracle, x, dtype)
    want, bound = ref.projection(value_of(x), ref.values(codes, scales, 320), dtype)
    got = project(device, queue, dtype, x, codes, scales, rows, 320, 70)
    plain = np.isfinite(want)
    assert np.isnan(got[1]).all() and np.isnan(got[:, 5]).all() and np.isnan(got[:, 69]).all()
    assert not np.isfinite(got[2]).any()
    assert np.array_equal(plain, np.isfinite(got))
    close(got[plain], want[plain], bound[plain])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,inputs,outputs,shift,position", [(40, 12500, 70, 0, None), (5, 8330, 50, 1, None), (3, 12288, 20, 1, 2),
                                                                (70, 416, 130, 1, 4), (21, 4096, 40, 0, 1), (150, 1056, 1100, 0, None),
                                                                (33, 1, 1, 0, None), (4, 12320, 33, 1, None)])
def test_projection_other_forms(oracle, device, queue, dtype, rows, inputs, outputs, shift, position):
    """Long rows in many, scales that are no whole words in every form, one input, both sides of the rules."""
    rng = np.random.default_rng(rows + inputs)
    x = stored(oracle, rng.standard_normal((rows, inputs)), dtype)
    codes, scales = packed_random(rng, (outputs, inputs), inputs ** -0.5)
    want, bound = ref.projection(value_of(x), ref.values(codes, scales, inputs), dtype)
    close(project(device, queue, dtype, x, codes, scales, rows, inputs, outputs, shift, position), want, bound)


def test_projection_refuses_too_many_outputs(device, queue):
    room = device.allocate(1 << 16)
    at = room.ptr()
    for rows, inputs, outputs in ((1, 16384, 1 << 30), (1 << 30, 64, 1 << 30), ((1 << 30) + 1, 64, 1), (1, 64, (1 << 30) + 1)):
        with pytest.raises(_lib.DolittleError, match="too (large|many)"):
            _lib.call("dl_projection_fp4", queue.handle, 1, at, at, at, at, rows, inputs, outputs, None)


def test_projection_same_bits(oracle, device, queue):
    rng = np.random.default_rng(2)
    x = stored(oracle, rng.standard_normal((4, 4096)), "bf16")
    codes, scales = packed_random(rng, (200, 4096))
    first = project(device, queue, "bf16", x, codes, scales, 4, 4096, 200)
    assert np.array_equal(first, project(device, queue, "bf16", x, codes, scales, 4, 4096, 200))


# ------------------------------------------------------------------ attention
class Problem:
    """Operands of one attention call; rows past a length are NaN groups, the output and the workspace garbage."""

    def __init__(self, oracle, dtype, batch, rows, capacity, heads, lengths, window=0, sinks=0, seed=0, spread=1.0):
        rng = np.random.default_rng(seed * 1009 + batch * 31 + rows * 7 + capacity + window)
        qh, kvh, w = heads
        self.dtype, self.lengths, self.window, self.sinks = dtype, np.array(lengths, np.uint64), window, sinks
        self.shape = BatchShape(batch, rows, qh, kvh, w, capacity)
        self.q = stored(oracle, rng.standard_normal((batch, rows, qh, w)) * spread, dtype)
        self.kc, self.ks = packed_random(rng, (batch, kvh, capacity, w), spread)
        self.vc, self.vs = packed_random(rng, (batch, kvh, capacity, w))
        for b in range(batch):
            n = min(int(self.lengths[b]), capacity)
            self.kc[b, :, n:], self.vc[b, :, n:] = 0xA7, 0x5F
            self.ks[b, :, n:], self.vs[b, :, n:] = 255, 255
        self.scale = np.float32(1.0 / np.sqrt(w))

    def run(self, device, queue, shift=0):
        held = [up(device, queue, a, s) for a, s in ((self.q, shift), (self.kc, 0), (self.ks, shift), (self.vc, 0), (self.vs, shift))]
        q, kc, ks, vc, vs = (at for _, at in held)
        lengths, scale = up(device, queue, self.lengths), up(device, queue, np.array([self.scale]))
        room = attention_workspace_bytes(self.shape, self.window, self.sinks)
        work = device.upload_array(queue, np.full(room + 64, 0xFF, np.uint8))
        out = Room(device, queue, self.q.size, self.q.dtype, shift)
        cache = CacheAddresses(kc, ks, vc, vs)
        _lib.call("dl_attention_fp4", queue.handle, CODE[self.dtype], C.byref(self.shape), q, C.byref(cache), lengths[1],
                  self.window, self.sinks, out.at, scale[1], work.ptr(), room)
        got = out.read().reshape(self.q.shape)
        assert np.all(queue.read(work, np.uint8, 64, room) == 0xFF)
        return got

    def want(self):
        w = self.shape.width
        return ref.attention(value_of(self.q), ref.values(self.kc, self.ks, w), ref.values(self.vc, self.vs, w), self.lengths,
                             float(self.scale), self.window, self.sinks, self.dtype)

    def check(self, device, queue, **more):
        want, bound = self.want()
        close(value_of(self.run(device, queue, **more)), want, bound)


HEADS = [(4, 1, 128), (8, 2, 64), (3, 3, 80), (8, 1, 256), (10, 2, 96), (2, 1, 32), (2, 2, 200), (5, 1, 7), (20, 1, 128), (2, 1, 130)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("rows,window,sinks", [(1, 0, 0), (1, 40, 3), (5, 0, 0), (9, 17, 2)])
def test_attention(oracle, device, queue, dtype, heads, rows, window, sinks):
    Problem(oracle, dtype, 3, rows, 301, heads, [301, 130, rows], window, sinks).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths", [[0, 1, 2], [3, 32, 33], [31, 64, 96], [200, 127, 129], [1000, 128, 0]])
@pytest.mark.parametrize("rows", [1, 3])
def test_attention_lengths(oracle, device, queue, dtype, lengths, rows):
    """Empty and full caches, lengths below the new rows (rows that see nothing are zeros), lengths past the capacity."""
    Problem(oracle, dtype, 3, rows, 200, (4, 2, 64), lengths).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 0), (32, 4), (33, 40), (64, 200), (100, 1000), (299, 1), (300, 0), (5, 64),
                                          (1 << 50, 3)])
@pytest.mark.parametrize("rows", [1, 4, 40])
def test_attention_windows(oracle, device, queue, dtype, window, sinks, rows):
    """Windows that begin inside the sinks, at a step's border and past the cache; rows whose windows part."""
    Problem(oracle, dtype, 2, rows, 300, (4, 2, 64), [300, 171], window, sinks).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,capacity,heads,window", [(70, 300, (4, 1, 128), 0), (130, 300, (4, 2, 64), 0), (150, 400, (2, 2, 96), 60),
                                                        (65, 260, (4, 2, 256), 0), (90, 200, (3, 1, 80), 33)])
def test_attention_chunks(oracle, device, queue, dtype, rows, capacity, heads, window):
    Problem(oracle, dtype, 2, rows, capacity, heads, [capacity, rows + 11], window, 2 if window else 0).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(4, 2, 104), (4, 1, 232), (2, 2, 128), (3, 1, 256)])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_rows_of_scale_words(oracle, device, queue, dtype, heads, rows):
    """Rows whose scales are whole words but whose last group is not full; lengths inside a step."""
    Problem(oracle, dtype, 3, rows, 333, heads, [333, 97, 71], seed=3).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [0, 3000])
def test_attention_long(oracle, device, queue, dtype, window):
    """Many ranges of one long cache, joined."""
    Problem(oracle, dtype, 1, 1, 20000, (4, 1, 128), [19977], window, 5).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_off_alignment(oracle, device, queue, dtype):
    Problem(oracle, dtype, 2, 3, 77, (4, 2, 128), [77, 40]).check(device, queue, shift=1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-30])
def test_attention_scales(oracle, device, queue, dtype, scale):
    p = Problem(oracle, dtype, 2, 3, 120, (4, 2, 64), [120, 60], 50, 2)
    p.scale = np.float32(scale)
    p.check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_large_scores(oracle, device, queue, dtype):
    """Scores that rise by far more than an exponential holds, in every order."""
    p = Problem(oracle, dtype, 2, 2, 256, (2, 1, 64), [256, 200], spread=6.0)
    p.ks[0, 0, :256] = np.minimum(p.ks[0, 0, :256].astype(int) + (np.arange(256) // 64)[:, None], 252)
    p.ks[1, 0, :200] = np.minimum(p.ks[1, 0, :200].astype(int) + (3 - np.arange(200) // 64)[:, None], 252)
    p.check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,window", [(1, 0), (6, 0), (6, 9), (80, 0), (80, 30)])
def test_attention_nan_groups(oracle, device, queue, dtype, rows, window):
    """NaN groups of keys and values reach the rows that see them, and no bit of any other row."""
    capacity, n = 160, 150
    plain = Problem(oracle, dtype, 1, rows, capacity, (4, 1, 128), [n], window, 2)
    first = plain.run(device, queue)
    p = Problem(oracle, dtype, 1, rows, capacity, (4, 1, 128), [n], window, 2)
    late = n - max(rows // 2, 1)  # the rows before it do not see it
    p.vs[0, 0, late, 1] = 255
    if window:
        p.ks[0, 0, 20, 3] = 255
        p.vs[0, 0, 21, 0] = 255
    p.check(device, queue)
    got = p.run(device, queue)
    touched = np.isnan(value_of(got))
    for i in range(rows):
        seen = ref.sight(n, rows, i, window, 2)
        if not {late, *((20, 21) if window else ())} & set(seen):
            assert np.array_equal(got[0, i], first[0, i])
        elif not (window and 20 in seen):
            # the value group's features alone, the others to the bit
            assert touched[0, i, :, 32:64].all() == (late in seen)
            assert np.array_equal(got[0, i, :, 64:], first[0, i, :, 64:])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_nan_query(oracle, device, queue, dtype):
    p = Problem(oracle, dtype, 1, 3, 90, (4, 2, 64), [90])
    nan = stored(oracle, [np.nan], dtype)[0]
    p.q[0, 1, 2, 5] = nan
    p.check(device, queue)


def test_attention_rows_alone_and_together(oracle, device, queue):
    """Same bits from the same call; hidden rows of a cache change none."""
    p = Problem(oracle, "bf16", 2, 5, 300, (8, 2, 128), [260, 33], 50, 4)
    first = p.run(device, queue)
    assert np.array_equal(first, p.run(device, queue))
    for b, n in enumerate((260, 33)):
        p.kc[b, :, n:], p.ks[b, :, n:], p.vc[b, :, n:], p.vs[b, :, n:] = 0x33, 120, 0x44, 130
    p.kc[0, :, 60:200], p.vc[0, :, 60:200] = 0x77, 0x77  # behind every window
    assert np.array_equal(first, p.run(device, queue))


# --------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(8, 2, 128), (4, 4, 64), (6, 3, 80), (2, 1, 256), (20, 10, 96), (2, 1, 2), (3, 3, 34)])
@pytest.mark.parametrize("rows,in_place,shift", [(1, True, 0), (1, False, 1), (7, True, 0), (7, False, 0)])
def test_append(oracle, device, queue, dtype, heads, rows, in_place, shift):
    qh, kvh, w = heads
    batch, capacity = 3, 21
    rng = np.random.default_rng(w + rows)
    lengths = np.array([0, 13, capacity - (rows // 2)], np.uint64)  # the last has no room for all
    positions = np.array([0, 1 << 20, 77], np.uint64)
    q, k, v = (stored(oracle, rng.standard_normal((batch, rows, h, w)), dtype) for h in (qh, kvh, kvh))
    codes, scales = packed_random(rng, (2, batch, kvh, capacity, w))
    shape = BatchShape(batch, rows, qh, kvh, w, capacity)
    held = [up(device, queue, a, shift) for a in (q, k, v)]
    caches = [Room(device, queue, a.size, np.uint8, s) for a, s in ((codes[0], 0), (scales[0], shift), (codes[1], 0), (scales[1], shift))]
    for room, a in zip(caches, (codes[0], scales[0], codes[1], scales[1])):
        queue.write(room.buffer, a, room.before)
    out = Room(device, queue, q.size, q.dtype, shift)
    n, p = up(device, queue, lengths), up(device, queue, positions)
    n_out, p_out = (n, p) if in_place else (up(device, queue, lengths * 0), up(device, queue, positions * 0))
    addresses = CacheAddresses(*(c.at for c in caches))
    _lib.call("dl_cache_append_fp4", queue.handle, CODE[dtype], C.byref(shape), held[0][1], held[1][1], held[2][1], out.at,
              C.byref(addresses), n[1], n_out[1], p[1], p_out[1], 1e6)
    at = positions[:, None] + np.arange(rows, dtype=np.uint64)
    want_q = ref.rotated(value_of(q), at)
    got_q = value_of(out.read().reshape(q.shape))
    assert np.array_equal(got_q, value_of(stored(oracle, want_q, dtype)))
    want_k, want_v = ref.quantized(ref.rotated(value_of(k), at).astype(np.float64)), ref.quantized(value_of(v))
    for b in range(batch):
        for i in range(rows):
            slot = int(lengths[b]) + i
            if slot < capacity:
                for c, (new_codes, new_scales) in enumerate((want_k, want_v)):
                    codes[c, b, :, slot], scales[c, b, :, slot] = new_codes[b, i], new_scales[b, i]
    for room, a in zip(caches, (codes[0], scales[0], codes[1], scales[1])):
        assert np.array_equal(room.read(), a.reshape(-1))
    assert np.array_equal(queue.read(n_out[0], np.uint64, batch), np.minimum(lengths + rows, capacity))
    assert np.array_equal(queue.read(p_out[0], np.uint64, batch), positions + rows)


def test_append_special_values(oracle, device, queue):
    """A NaN feature of a key makes NaN of its groups (both halves of the rotation), and of no other head or row."""
    x = np.ones((1, 2, 2, 128), np.float32)
    x[0, 1, 0, 3] = np.nan
    cache = Fp4Cache(device, queue, 1, 8, 2, 2, 128)
    row = up(device, queue, stored(oracle, x, "bf16"))
    rotated = device.allocate(x.size * 2)
    cache.append(row[0], row[0], row[0], rotated, 2)
    queue.drain()
    for scales, groups in ((cache.key_scales, [0, 2]), (cache.value_scales, [0])):
        nan = queue.read(scales, np.uint8, 2 * 8 * 4).reshape(2, 8, 4)[:, :2] == 255
        assert np.argwhere(nan).tolist() == [[0, 1, g] for g in groups]


# ---------------------------------------------------- a decode step of all of them
def decode_step(dims, device, queue, cache, weights, buffers, dtype, rows):
    """Query, key and value projections, append, attention and output projection."""
    for name in ("q", "k", "v"):
        weights[name].project(buffers["x"], buffers[name], dims["batch"] * rows, dtype)
    cache.append(buffers["q"], buffers["k"], buffers["v"], buffers["rotated"], rows)
    cache.attend(buffers["rotated"], buffers["attended"], rows)
    weights["o"].project(buffers["attended"], buffers["y"], dims["batch"] * rows, dtype)


class Layer:
    """An attention layer whose weights and cache are held in 4 bits."""

    def __init__(self, oracle, device, queue, dtype, batch, capacity, window, sinks, most_rows, seed=3):
        self.oracle, self.device, self.queue, self.dtype = oracle, device, queue, dtype
        self.dims = {"batch": batch, "qh": 8, "kvh": 2, "w": 64, "hidden": 320}
        d = self.dims
        rng = np.random.default_rng(seed)
        widths = {"q": (d["qh"] * d["w"], d["hidden"]), "k": (d["kvh"] * d["w"], d["hidden"]), "v": (d["kvh"] * d["w"], d["hidden"]),
                  "o": (d["hidden"], d["qh"] * d["w"])}
        self.weights, self.values = {}, {}
        for name, (outputs, inputs) in widths.items():
            w = stored(oracle, rng.standard_normal((outputs, inputs)) * inputs ** -0.5, dtype)
            held = up(device, queue, w)
            self.weights[name] = Fp4Weight(device, queue, outputs, inputs)
            self.weights[name].quantize(held[0], dtype)
            queue.drain()
            self.values[name] = ref.values(*ref.quantized(value_of(w)), inputs)
        self.cache = Fp4Cache(device, queue, batch, capacity, d["qh"], d["kvh"], d["w"], dtype, window=window, sinks=sinks)
        n = batch * most_rows
        sizes = {"x": d["hidden"], "q": d["qh"] * d["w"], "k": d["kvh"] * d["w"], "v": d["kvh"] * d["w"], "rotated": d["qh"] * d["w"],
                 "attended": d["qh"] * d["w"], "y": d["hidden"]}
        self.buffers = {name: device.allocate(n * size * SIZE[dtype]) for name, size in sizes.items()}
        self.sizes = sizes

    def step(self, rows):
        decode_step(self.dims, self.device, self.queue, self.cache, self.weights, self.buffers, self.dtype, rows)

    def read(self, name, rows):
        n = self.dims["batch"] * rows
        return self.queue.read(self.buffers[name], storage(self.dtype), n * self.sizes[name]).reshape(n, -1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_prompt_and_decode_steps(oracle, device, queue, dtype, window, sinks):
    """A prompt chunk and decode steps through projections, append and attention: every stage against its formula
    on the inputs that the stage before it left."""
    batch = 2
    layer = Layer(oracle, device, queue, dtype, batch, 64, window, sinks, 30)
    d, rng = layer.dims, np.random.default_rng(9)
    keys, values = np.zeros((batch, d["kvh"], 64, d["w"])), np.zeros((batch, d["kvh"], 64, d["w"]))
    length = 0
    for rows in (30, 1, 1, 3, 1):
        x = stored(oracle, rng.standard_normal((batch * rows, d["hidden"])), dtype)
        queue.write(layer.buffers["x"], x)
        layer.step(rows)
        queue.drain()
        got = {n: layer.read(n, rows) for n in layer.sizes}
        for name in ("q", "k", "v"):
            want, bound = ref.projection(value_of(x), layer.values[name], dtype)
            close(value_of(got[name]), want, bound)
        at = length + np.arange(rows, dtype=np.uint64)[None].repeat(batch, 0)
        split = lambda name, heads: value_of(got[name]).reshape(batch, rows, heads, d["w"])  # noqa: E731
        turned = ref.rotated(split("q", d["qh"]), at)
        assert np.array_equal(split("rotated", d["qh"]), value_of(stored(oracle, turned, dtype)))
        new_k = ref.values(*ref.quantized(ref.rotated(split("k", d["kvh"]), at).astype(np.float64)), d["w"])
        new_v = ref.values(*ref.quantized(split("v", d["kvh"])), d["w"])
        keys[:, :, length:length + rows], values[:, :, length:length + rows] = new_k.transpose(0, 2, 1, 3), new_v.transpose(0, 2, 1, 3)
        length += rows
        assert layer.cache.used == [length] * batch
        want, bound = ref.attention(split("rotated", d["qh"]), keys, values, [length] * batch, float(np.float32(0.125)), window, sinks, dtype)
        close(split("attended", d["qh"]), want, bound)
        want, bound = ref.projection(value_of(got["attended"]), layer.values["o"], dtype)
        close(value_of(got["y"]), want, bound)
    with pytest.raises(LengthError):
        layer.step(64)


def test_steps_replayed_from_graphs(oracle, device, queue):
    """A decode step recorded once into a sequence's graphs and replayed nine times, twice, with eager work between:
    the bits of the same steps submitted one by one."""
    steps, batch = 9, 3
    eager, replayed = (Layer(oracle, device, queue, "bf16", batch, 200, 12, 2, 1) for _ in range(2))
    x = stored(oracle, np.random.default_rng(4).standard_normal((batch, 320)), "bf16")
    for layer in (eager, replayed):  # the workspace is there before the step is recorded
        queue.write(layer.buffers["x"], x)
        layer.step(1)
    queue.drain()
    ids = device.upload_array(queue, np.arange(steps, dtype=np.uint32))
    token = device.allocate(4)
    for turn in range(2):
        handle = C.c_void_p()
        _lib.call("dl_sequence_create", queue.handle, steps, 0, 1, 1, C.byref(handle))
        try:
            _lib.call("dl_sequence_begin", handle, None, None, token.ptr(), 4, ids.ptr(), steps * 4, None, None, None, None)
            for stage in range(4):
                _lib.call("dl_sequence_begin_stage", handle, stage)
                if stage == 0:
                    replayed.step(1)
                if stage == 3:
                    _lib.call("dl_sequence_begin_selection", handle)
                _lib.call("dl_sequence_end_stage", handle)
            _lib.call("dl_sequence_complete", handle)
            _lib.call("dl_sequence_start", handle)
            _lib.call("dl_sequence_drain", handle)
        finally:
            _lib.call("dl_sequence_destroy", handle)
        for _ in range(steps):
            eager.step(1)
        queue.drain()
        for name in ("rotated", "attended", "y"):
            assert np.array_equal(replayed.read(name, 1), eager.read(name, 1))
        for a, b in zip(replayed.cache._buffers, eager.cache._buffers):  # [batch][kv_heads][capacity][...]
            a, b = (queue.read(x, np.uint8, x.nbytes).reshape(batch, 2, 200, -1)[:, :, :1 + steps * (turn + 1)] for x in (a, b))
            assert np.array_equal(a, b)
        assert list(queue.read(replayed.cache.lengths, np.uint64, batch)) == [1 + steps * (turn + 1)] * batch
