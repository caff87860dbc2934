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
