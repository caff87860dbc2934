"""The operations over 4-bit storage at sizes whose launches differ from those of
test_gpu_fp4.py, against the same formulas in 64 bits."""
import numpy as np
import pytest

import fp4_reference as ref
from test_gpu_fp4 import Problem, close, value_of

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
