"""The operations over 4-bit storage at sizes whose launches differ from those of
test_gpu_fp4.py, against the same formulas in 64 bits."""
import numpy as np
import pytest

import fp4_reference as ref
from dolittle_amd.batch import BatchShape
from dolittle_amd.fp4 import attention_workspace_bytes
from test_gpu_fp4 import Problem, close, packed_random, project, stored, value_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("capacity,lengths,window", [(64, [50], 0), (20000, [900], 0), (20000, [900], 300)])
def test_attention_of_more_rows_than_a_join_takes(oracle, device, queue, dtype, capacity, lengths, window):
    """2^23 heads of rows and more: rows before the first slot are zeros, the last ones the formula's."""
    rows, last = 262200, 40
    p = Problem(oracle, dtype, 1, rows, capacity, (32, 2, 4), lengths, window, 3 if window else 0)
    assert rows * 32 > 1 << 23
    got = value_of(p.run(device, queue))
    assert not got[:, :rows - lengths[0]].any()
    w = p.shape.width
    want, bound = ref.attention(value_of(p.q[:, -last:]), ref.values(p.kc, p.ks, w), ref.values(p.vc, p.vs, w), p.lengths,
                                float(p.scale), p.window, p.sinks, dtype)
    close(got[:, -last:], want, bound)


# ------------------------------------------- projections whose stages go round the ring
DISTINCT = 509  # outputs that repeat: no multiple of a tile or a set


def weights(rng, inputs):
    """Codes and scales of DISTINCT outputs, random to the bit; zeros past the width."""
    groups = ref.groups_of(inputs)
    codes = rng.integers(0, 256, (DISTINCT, groups * 16), dtype=np.uint8)
    codes[:, (inputs + 1) // 2:] = 0
    if inputs % 2:
        codes[:, inputs // 2] &= 15
    return codes.reshape(DISTINCT, groups, 16), rng.integers(114, 124, (DISTINCT, groups), dtype=np.uint8)


def stages(inputs, outputs):
    """Stages of a workgroup of the staged projection and of the last, by its rule for sets of 2048 groups."""
    groups = ref.groups_of(inputs)
    row = 32 if groups <= 32 else 64 if groups <= 64 else 128
    sets = -(-outputs // (2048 // row))
    each = -(-sets // 256)
    blocks = -(-groups // 128)
    return each * blocks, (sets - (-(-sets // each) - 1) * each) * blocks


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,inputs,outputs", [
    # whole words of scales; rows of whole pieces, then not
    (2, 1024, 70001), (1, 1021, 54321), (3, 2048, 40001), (2, 2045, 30003), (2, 4096, 20005), (16, 4096, 61000), (1, 4093, 28711),
    (2, 8192, 16500), (5, 8189, 13000), (1, 12288, 16500), (3, 12285, 13001),
    # odd numbers of scales
    (3, 992, 50001), (2, 2016, 41003), (5, 4064, 24601), (1, 8160, 12601), (4, 12256, 16501),
    # two row tiles
    (18, 4096, 16405), (20, 8192, 13003)])
def test_projection_of_many_stages(oracle, device, queue, dtype, rows, inputs, outputs):
    of_each, of_last = stages(inputs, outputs)
    assert of_each >= 4 and of_last >= 1
    rng = np.random.default_rng(rows + inputs + outputs)
    x = stored(oracle, rng.standard_normal((rows, inputs)), dtype)
    codes, scales = weights(rng, inputs)
    want, bound = ref.projection(value_of(x), ref.values(codes, scales, inputs), dtype)
    at = np.arange(outputs) % DISTINCT
    got = project(device, queue, dtype, x, codes[at], scales[at], rows, inputs, outputs)
    close(got, want[:, at], bound[:, at])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("inputs,outputs", [(1000, 66001), (2048, 33001), (4096, 20005), (8192, 16500), (12288, 13001)])
def test_projection_of_many_stages_off_alignment(oracle, device, queue, dtype, inputs, outputs):
    assert stages(inputs, outputs)[0] >= 4
    rng = np.random.default_rng(inputs)
    x = stored(oracle, rng.standard_normal((2, inputs)), dtype)
    codes, scales = weights(rng, inputs)
    want, bound = ref.projection(value_of(x), ref.values(codes, scales, inputs), dtype)
    at = np.arange(outputs) % DISTINCT
    close(project(device, queue, dtype, x, codes[at], scales[at], 2, inputs, outputs, 1, 1), want[:, at], bound[:, at])


def test_stages_of_the_cases():
    """All remainders of a workgroup's stages by the ring's three, first and last workgroups."""
    sizes = ((1024, 70001), (1021, 54321), (2048, 40001), (4096, 20005), (4096, 61000), (4093, 28711), (992, 50001), (4064, 24601))
    found = [stages(*size) for size in sizes]
    assert {each % 3 for each, _ in found} == {0, 1, 2} and {last % 3 for _, last in found} == {0, 1, 2}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,inputs,outputs,shift", [(20, 12500, 33, 0), (17, 12320, 50, 1), (6, 16000, 20, 0)])
def test_projection_of_long_rows_in_tiles(oracle, device, queue, dtype, rows, inputs, outputs, shift):
    """More rows than one tile of the kernel for more than 12,288 inputs."""
    rng = np.random.default_rng(rows)
    x = stored(oracle, rng.standard_normal((rows, inputs)), dtype)
    codes, scales = packed_random(rng, (outputs, inputs), inputs ** -0.5)
    want, bound = ref.projection(value_of(x), ref.values(codes, scales, inputs), dtype)
    close(project(device, queue, dtype, x, codes, scales, rows, inputs, outputs, shift), want, bound)


# ---------------------------------------- attention whose steps go round the ring
class Heads(Problem):
    """Seven KV heads of a few query heads, over and over: so many tasks that each has one range of all steps."""
    SEVENS = 25

    def __init__(self, oracle, dtype, batch, rows, capacity, group, width, lengths, window=0, sinks=0, rising=0):
        super().__init__(oracle, dtype, batch, rows, capacity, (7 * group, 7, width), lengths, window, sinks)
        if rising:  # scores double every `rising` keys: the maximum is raised far behind the first steps
            up = (np.arange(capacity) // rising)[None, None, :, None]
            self.ks = np.where(self.ks == 255, 255, np.minimum(self.ks.astype(int) + up, 250)).astype(np.uint8)

    def check(self, device, queue, shift=0):
        want, bound = self.want()
        small = self.q, self.kc, self.ks, self.vc, self.vs
        n = self.SEVENS
        self.q = np.tile(self.q, (1, 1, n, 1))
        self.kc, self.vc = (np.tile(x, (1, n, 1, 1, 1)) for x in (self.kc, self.vc))
        self.ks, self.vs = (np.tile(x, (1, n, 1, 1)) for x in (self.ks, self.vs))
        s = self.shape
        self.shape = BatchShape(s.batch, s.rows, s.query_heads * n, s.kv_heads * n, s.width, s.capacity)
        assert attention_workspace_bytes(self.shape, self.window, self.sinks) == 0  # one range
        seen = min(max(self.lengths), self.window + s.rows if self.window else s.capacity)
        assert seen >= 8 * 4 * 32  # eight steps of each wavefront
        got = self.run(device, queue, shift)
        parts = got.reshape(s.batch, s.rows, n, s.query_heads, s.width)
        assert np.array_equal(parts, np.broadcast_to(parts[:, :, :1], parts.shape), equal_nan=got.dtype == np.float32)
        close(value_of(parts[:, :, 0]), want, bound)
        self.q, self.kc, self.ks, self.vc, self.vs = small


WIDTHS = [64, 40, 128, 96, 256, 200]  # tiles of 64, 128 and 256 features, scales in words and not


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("window,sinks,rising,shift", [(0, 0, 0, 0), (1100, 40, 0, 0), (0, 0, 200, 0), (1100, 3, 150, 1)])
def test_attention_of_many_steps(oracle, device, queue, dtype, width, window, sinks, rising, shift):
    Heads(oracle, dtype, 3, 1, 1500, 2, width, [1500, 1227, 1029], window, sinks, rising).check(device, queue, shift)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("window,sinks,rising", [(0, 0, 0), (1000, 5, 150)])
def test_attention_of_many_steps_in_chunks(oracle, device, queue, dtype, width, window, sinks, rising):
    """Two tiles of rows a wavefront in BF16 storage."""
    Heads(oracle, dtype, 3, 70, 1200, 1, width, [1200, 1111, 90], window, sinks, rising).check(device, queue)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("width", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 70])
def test_attention_of_many_steps_with_nan_groups(oracle, device, queue, dtype, width, rows):
    p = Heads(oracle, dtype, 3, rows, 1200, 1, width, [1200, 1111, 1050])
    p.vs[0, 3, 700, 1] = 255       # a value group that every row sees
    p.ks[1, 5, 600, 0] = 255       # a key
    p.vs[2, 1, 1050 - rows // 2 - 1, 0] = 255  # seen by the later rows alone
    p.check(device, queue)
