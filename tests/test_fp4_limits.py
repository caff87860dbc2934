"""Limits of the attention over 4-bit caches (include/dolittle_hip.h, dl_attention_fp4):
calls of many rows that need no join, or can do without one, are no larger than the
launch itself may be.  Nothing here reaches a device."""
import pytest

from dolittle_amd import LengthError
from dolittle_amd.batch import BatchShape
from dolittle_amd.fp4 import attention_workspace_bytes
from test_fp4_host import attend, library  # noqa: F401
from dolittle_amd import InvalidArgument

MOST = (1 << 23) - 8


@pytest.mark.parametrize("window", [0, 511])
@pytest.mark.parametrize("shape", [
    (1, 1 << 20, 16, 2, 128, 2048),        # a single range
    (8, 32768, 64, 8, 128, 32768),         # long prompts of a batch
    (1, 1 << 19, 32, 8, 128, 1 << 19),
    (64, 4096, 64, 8, 128, 4096),
    (1, (1 << 24) - 16, 1, 1, 2, 1 << 30),  # the longest cache
    (1, 16 * MOST // 8 >> 8, 256, 1, 64, 4096),  # the most tiles: heads count in eights
])
def test_many_rows_are_taken(shape, window):
    s = BatchShape(*shape)
    assert attention_workspace_bytes(s, window, 4) >= 0
    with pytest.raises(InvalidArgument, match="null queue"):
        attend(s, window=window, sinks=4)


@pytest.mark.parametrize("batch,kv_heads", [(64, 64), (1 << 12, 1 << 10), (1 << 18, 8)])
def test_long_caches_of_many_heads_are_taken(batch, kv_heads):
    """Ranges are cut to what a launch has room for."""
    s = BatchShape(batch, 1, kv_heads, kv_heads, 2, 1 << 30)
    with pytest.raises(InvalidArgument, match="null queue"):
        attend(s)


@pytest.mark.parametrize("shape", [
    (1, (16 * MOST // 8 >> 8) + 16, 256, 1, 64, 4096),  # one tile of 16 rows too many would need more
    (1, 1 << 24, 64, 1, 64, 4096),
    (1 << 20, 1, 8, 8, 64, 32),
])
def test_more_tiles_than_a_launch_has_are_refused(shape):
    with pytest.raises(LengthError, match="too many row tiles"):
        attention_workspace_bytes(BatchShape(*shape))
