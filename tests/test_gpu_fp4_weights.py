"""Attention over 4-bit caches where values cancel: keys come in pairs whose weights
differ by a few hundredths and whose values are each other's negatives, so the output
is the weights' difference.  A weight rounded to BF16 alone (2^-8) would be most of it.

Bound.  BF16 storage holds a weight as two BF16 values, the second of what the first
leaves: off by at most 2^-8 of 2^-8, 2^-16 of the weight.  All else is as for FP32
storage (fp4_reference.attention, whose three products a weight are at least as many
terms), and the result is rounded once, 2^-8."""
import numpy as np
import pytest

import fp4_reference as ref
from dolittle_amd.fp4 import attention_workspace_bytes
from test_gpu_fp4 import Problem, close, value_of

pytestmark = pytest.mark.gpu


def paired(oracle, *args, **more):
    """A problem of such pairs; its lengths are even."""
    p = Problem(oracle, *args, **more)
    for b, n in enumerate(p.lengths):
        n = int(n)
        for codes, scales in ((p.kc, p.ks), (p.vc, p.vs)):
            codes[b, :, 1:n:2], scales[b, :, 1:n:2] = codes[b, :, 0:n:2], scales[b, :, 0:n:2]
        p.kc[b, :, 1:n:2, 0, 0] ^= 1  # the first feature by half of a step of its code
        p.vc[b, :, 1:n:2] ^= 0x88
    return p


def want(p):
    w = p.shape.width
    q, key, value = value_of(p.q), ref.values(p.kc, p.ks, w), ref.values(p.vc, p.vs, w)
    rest = p.lengths, float(p.scale), p.window, p.sinks, "f32"
    out, bound = ref.attention(q, key, value, *rest)
    if p.dtype == "bf16":
        size, _ = ref.attention(q, key, np.abs(value), *rest)
        bound = bound + 1.01 * (2.0 ** -16 * size + 2.0 ** -8 * np.abs(out))
    return out, bound


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads", [(4, 2, 64), (8, 1, 128), (3, 3, 80), (4, 1, 256)])
@pytest.mark.parametrize("rows,window,sinks", [(1, 0, 0), (2, 8, 2), (90, 0, 0), (90, 30, 4)])
def test_attention_of_cancelling_values(oracle, device, queue, dtype, heads, rows, window, sinks):
    p = paired(oracle, dtype, 4, rows, 300, heads, [2, 6, 90, 300], window, sinks)
    close(value_of(p.run(device, queue)), *want(p))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_of_cancelling_values_over_ranges(oracle, device, queue, dtype):
    p = paired(oracle, dtype, 2, 1, 4000, (4, 1, 128), [4000, 1030])
    close(value_of(p.run(device, queue)), *want(p))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,heads,n,second,largest", [
    (1, 1, 300, 170, 10),    # joined with another wavefront's
    (1, 1, 300, 170, 290),   # with another range's
    (8, 64, 420, 170, 300),  # raised in the same wavefront
])
def test_a_weight_far_below_the_largest(oracle, device, queue, dtype, batch, heads, n, second, largest):
    """The largest score is 88 and its value 0; that of the second, 8.25, is 1, so the output is exp(-79.75).  All other
    scores are 0: the second key is counted from their maximum, which lies e^-88 below the largest, under 2^-126."""
    p = Problem(oracle, dtype, batch, 1, n, (heads, heads, 32), [n] * batch)
    p.kc[:], p.vc[:], p.ks[:], p.vs[:] = 0, 0, 127, 127
    p.kc[:, :, second, 0, 0], p.kc[:, :, largest, 0, 0] = 7, 6  # 6 and 4
    p.ks[:, :, largest] = 131
    p.vc[:, :, second] = 0x22
    p.q[:] = 0
    p.q[..., 0] = 0x3fb0 if dtype == "bf16" else 1.375
    p.scale = np.float32(1)
    assert (attention_workspace_bytes(p.shape) == 0) == (heads == 64)
    out, bound = want(p)
    assert np.allclose(out, np.exp(-79.75), rtol=1e-6) and bound.max() < 0.1 * out.min()
    close(value_of(p.run(device, queue)), out, bound)
