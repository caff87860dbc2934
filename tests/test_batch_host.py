"""Argument checks of the batch attention and cache operations
(include/dolittle_hip.h, dl_batch_shape): every refusal happens before a
device is touched, so none of these calls needs one."""
import ctypes as C
import os

import pytest

from dolittle_amd import InvalidArgument, LengthError, _lib
from dolittle_amd.batch import BatchShape, workspace_bytes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module", autouse=True)
def library():
    if not os.path.exists(_lib.LIBRARY):
        from dolittle_amd import build
        build.build()
    _lib.load()


def shape(batch=2, rows=1, query_heads=8, kv_heads=2, width=64, capacity=32):
    return BatchShape(batch, rows, query_heads, kv_heads, width, capacity)


P = C.c_void_p(4096)  # an address that no check dereferences


def attention(name, s, dtype=1, prefix=5, room=None, **null):
    def p(n):
        return None if n in null else P
    room = workspace_bytes(name, s, prefix) if room is None else room
    args = [p("query"), p("prefix_key"), p("prefix_value"), prefix, p("key"), p("value"), p("lengths")]
    if name == "dl_attention_weighted":
        args += [p("weights"), p("weights_out")]
    work = C.c_void_p(null["work"]) if "work" in null else P
    _lib.call(name, None, dtype, C.byref(s), *args, p("output"), p("scale"), work, room)


def append(s, dtype=1, theta=1e6, missing=None):
    _lib.call("dl_cache_append", None, dtype, C.byref(s), *[None if i == missing else P for i in range(12)], theta)


def evict(s, dtype=1, budget=8, sinks=1, recent=2, missing=None, work=4096, room=None):
    room = workspace_bytes("dl_cache_evict", s, budget) if room is None else room
    _lib.call("dl_cache_evict", None, dtype, C.byref(s), *[None if i == missing else P for i in range(8)], budget, sinks,
              recent, C.c_void_p(work) if work else None, room)


NAMES = ["dl_attention_shared", "dl_attention_weighted"]


@pytest.mark.parametrize("name", NAMES)
def test_complete_calls_reach_the_queue_check(name):
    with pytest.raises(InvalidArgument, match="null queue"):
        attention(name, shape())
    with pytest.raises(InvalidArgument, match="null queue"):
        attention(name, shape(), prefix=0, prefix_key=1, prefix_value=1)  # an empty prefix has no operands
    with pytest.raises(InvalidArgument, match="null queue"):
        append(shape())
    with pytest.raises(InvalidArgument, match="null queue"):
        evict(shape())


@pytest.mark.parametrize("field", ["batch", "rows", "query_heads", "kv_heads", "width", "capacity"])
def test_empty_shapes(field):
    for name in (*NAMES, "dl_cache_evict"):
        with pytest.raises(InvalidArgument):
            workspace_bytes(name, shape(**{field: 0}), 4)
    with pytest.raises(InvalidArgument):
        append(shape(**{field: 0}))
    with pytest.raises(InvalidArgument):
        evict(shape(**{field: 0}), room=1 << 20)


@pytest.mark.parametrize("name", NAMES)
def test_attention_refusals(name):
    with pytest.raises(InvalidArgument, match="multiple"):
        attention(name, shape(query_heads=7), room=1 << 30)
    for dtype in (0, 3, 7):
        with pytest.raises(InvalidArgument, match="storage type"):
            attention(name, shape(), dtype=dtype)
    for operand in ("query", "prefix_key", "prefix_value", "key", "value", "lengths", "output", "scale"):
        with pytest.raises(InvalidArgument, match="null"):
            attention(name, shape(), **{operand: 1})
    if name == "dl_attention_weighted":
        for operand in ("weights", "weights_out"):
            with pytest.raises(InvalidArgument, match="null"):
                attention(name, shape(), **{operand: 1})
    need = workspace_bytes(name, shape(), 5)
    with pytest.raises(LengthError, match="workspace"):
        attention(name, shape(), room=need - 1)
    for work in (0, 4097, 4104):
        with pytest.raises(InvalidArgument, match="workspace"):
            attention(name, shape(), work=work)
    for big in ({"width": 257}, {"capacity": (1 << 30) + 1}, {"batch": (1 << 20) + 1}, {"rows": (1 << 24) + 1},
                {"batch": 1 << 20, "rows": 1 << 12}, {"query_heads": 1 << 17, "kv_heads": 1 << 17},
                {"kv_heads": 1 << 16, "query_heads": 1 << 16, "width": 256 + 1}):
        with pytest.raises(LengthError):
            workspace_bytes(name, shape(**big), 5)
    with pytest.raises(LengthError):
        workspace_bytes(name, shape(), (1 << 30) + 1)
    with pytest.raises(InvalidArgument):
        _lib.call(name + "_bytes", C.byref(shape()), 5, None)
    with pytest.raises(InvalidArgument):
        _lib.call(name + "_bytes", None, 5, C.byref(C.c_uint64()))


def test_workspace_covers_what_is_written():
    """Eight bytes and a row per range, KV head and query row, and eight more
    per row for the weights."""
    s = shape(batch=3, rows=5, query_heads=12, kv_heads=4, width=80, capacity=700)
    rows = 3 * 5 * 3
    plain, weighted = (workspace_bytes(n, s, 1000) for n in NAMES)
    assert plain >= 2 * 4 * rows * (8 + 80 * 4)
    assert weighted - plain >= 4 * rows * 8


def test_workspace_of_the_weights():
    """The weights of up to 16 rows a KV head need their scores, those of more rows each row's maximum and sum;
    the attention alone needs neither."""
    def pieces(nbytes):
        return (nbytes + 255) // 256 * 256

    for rows, heads, extra in ((5, 3, lambda s: s.rows * 704 * 4), (16, 1, lambda s: s.rows * 704 * 4),
                               (6, 3, lambda s: s.rows * 8), (17, 1, lambda s: s.rows * 8)):
        s = shape(batch=3, rows=rows, query_heads=4 * heads, kv_heads=4, width=80, capacity=700)
        plain, weighted = (workspace_bytes(n, s, 1000) for n in NAMES)
        assert weighted - plain == pieces(extra(s) * 3 * 4 * heads), (rows, heads)


def test_append_refusals():
    for i in range(12):
        with pytest.raises(InvalidArgument, match="null operand"):
            append(shape(), missing=i)
    with pytest.raises(InvalidArgument, match="even"):
        append(shape(width=65))
    for theta in (0.0, -1.0, float("nan"), float("inf"), 1e301):
        with pytest.raises(InvalidArgument, match="theta"):
            append(shape(), theta=theta)
    with pytest.raises(InvalidArgument, match="storage type"):
        append(shape(), dtype=3)
    for big in ({"width": 4098}, {"batch": 65536}, {"query_heads": 1 << 16, "kv_heads": 1, "width": 512}):
        with pytest.raises(LengthError):
            append(shape(**big))


def test_evict_refusals():
    for i in range(8):
        with pytest.raises(InvalidArgument, match="null operand"):
            evict(shape(), missing=i)
    with pytest.raises(InvalidArgument, match="budget"):
        evict(shape(), budget=0, room=1 << 20)
    for sinks, recent in ((9, 0), (0, 9), (4, 5), ((1 << 64) - 1, 2), (1, (1 << 64) - 1)):
        with pytest.raises(InvalidArgument, match="exceed the budget"):
            evict(shape(), sinks=sinks, recent=recent)
    with pytest.raises(InvalidArgument, match="storage type"):
        evict(shape(), dtype=0)
    with pytest.raises(LengthError, match="workspace"):
        evict(shape(), room=workspace_bytes("dl_cache_evict", shape(), 8) - 1)
    for work in (0, 4098, 4100):
        with pytest.raises(InvalidArgument, match="workspace"):
            evict(shape(), work=work)
    with pytest.raises(LengthError):
        evict(shape(batch=40000))


def test_evict_workspace_follows_the_most_rows_that_can_move():
    for budget, most in ((1, 1), (8, 8), (16, 16), (31, 1), (32, 0), (1000, 0)):
        assert workspace_bytes("dl_cache_evict", shape(), budget) >= 4 * 4 * 2 * most
    assert workspace_bytes("dl_cache_evict", shape(capacity=1 << 20), 1 << 20) < 256  # nothing can move


def test_evict_workspace_refuses_what_the_eviction_refuses():
    with pytest.raises(LengthError, match="sequences"):
        workspace_bytes("dl_cache_evict", shape(batch=40000), 8)
    assert workspace_bytes("dl_cache_evict", shape(batch=65535, kv_heads=1), 8) > 0


def test_an_outgrown_workspace_stays_allocated():
    """Work recorded into a graph with the first workspace still writes to it
    after a later call needed more."""
    from dolittle_amd.batch import BatchCache

    class Buffer:
        freed = False

        def __init__(self, nbytes):
            self.nbytes = nbytes

        def ptr(self):
            return id(self)

        def free(self):
            self.freed = True

    class Owner:
        made = []

        def allocate(self, nbytes):
            self.made.append(Buffer(nbytes))
            return self.made[-1]

        def drain(self):
            pass

    cache = BatchCache.__new__(BatchCache)
    cache.device = cache.queue = owner = Owner()
    cache._work = []
    kept = [cache._workspace(need) for need in (100, 50, 101, 200, 1000)]
    assert [room for _, room in kept] == [100, 100, 200, 200, 1000]
    assert len(owner.made) == 3 and not any(b.freed for b in owner.made)
