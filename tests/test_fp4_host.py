"""Argument checks of the operations over 4-bit storage (include/dolittle_hip.h,
dl_fp4_cache): every refusal happens before a device is touched.  And the test
oracle's own rounding against the borders between neighbouring codes."""
import ctypes as C
import os

import numpy as np
import pytest

import fp4_reference as ref
from dolittle_amd import InvalidArgument, LengthError, _lib
from dolittle_amd.batch import BatchShape
from dolittle_amd.fp4 import CacheAddresses, Fp4Cache, Fp4Weight, attention_workspace_bytes, row_bytes


@pytest.fixture(scope="module", autouse=True)
def library():
    if not os.path.exists(_lib.LIBRARY):
        from dolittle_amd import build
        build.build()
    _lib.load()


P = C.c_void_p(4096)  # an address that no check dereferences


def shape(batch=2, rows=1, query_heads=8, kv_heads=2, width=64, capacity=32):
    return BatchShape(batch, rows, query_heads, kv_heads, width, capacity)


def cache(missing=None, at=None, address=0):
    names = ("key_codes", "key_scales", "value_codes", "value_scales")
    return CacheAddresses(*(None if n == missing else address if n == at else 4096 for n in names))


def pick(missing, *names):
    return [None if n == missing else P for n in names]


def quantize(dtype=1, rows=4, width=64, missing=None, codes=4096, name="dl_fp4_quantize"):
    x, s = pick(missing, "values", "scales")
    c = None if missing == "codes" else C.c_void_p(codes)
    args = (x, c, s) if name == "dl_fp4_quantize" else (c, s, x)
    _lib.call(name, None, dtype, *args, rows, width)


def project(dtype=1, rows=2, inputs=64, outputs=32, missing=None, codes=4096):
    x, s, y = pick(missing, "input", "scales", "output")
    _lib.call("dl_projection_fp4", None, dtype, x, None if missing == "codes" else C.c_void_p(codes), s, y, rows, inputs,
              outputs, None)


def append(s, dtype=1, theta=1e6, missing=None, held=None):
    q, k, v, out, n, n_out, p, p_out = pick(missing, "query", "key", "value", "query_out", "lengths", "lengths_out",
                                            "positions", "positions_out")
    held = held if held is not None else cache(missing)
    _lib.call("dl_cache_append_fp4", None, dtype, C.byref(s) if s else None, q, k, v, out,
              None if missing == "cache" else C.byref(held), n, n_out, p, p_out, theta)


def attend(s, dtype=1, window=0, sinks=0, missing=None, held=None, work=4096, room=None):
    q, n, out, scale = pick(missing, "query", "lengths", "output", "scale")
    held = held if held is not None else cache(missing)
    room = attention_workspace_bytes(s, window, sinks) if room is None else room
    _lib.call("dl_attention_fp4", None, dtype, C.byref(s) if s else None, q, None if missing == "cache" else C.byref(held), n,
              window, sinks, out, scale, C.c_void_p(work) if work else None, room)


def test_complete_calls_reach_the_queue_check():
    for call in (quantize, lambda: quantize(name="dl_fp4_values"), project, lambda: append(shape()), lambda: attend(shape()),
                 lambda: attend(shape(), window=5, sinks=2), lambda: project(inputs=1, outputs=1, rows=1)):
        with pytest.raises(InvalidArgument, match="null queue"):
            call()


def test_bytes():
    assert row_bytes(3, 64) == (3 * 2 * 16, 3 * 2)
    assert row_bytes(1, 1) == (16, 1)
    assert row_bytes(7, 1000) == (7 * 32 * 16, 7 * 32)
    for rows, width in ((0, 4), (4, 0)):
        with pytest.raises(InvalidArgument):
            row_bytes(rows, width)
    with pytest.raises(LengthError):
        row_bytes(1 << 41, 4)
    with pytest.raises(InvalidArgument):
        _lib.call("dl_fp4_bytes", 4, 4, None, None)


@pytest.mark.parametrize("name", ["dl_fp4_quantize", "dl_fp4_values"])
def test_row_refusals(name):
    for bad in (dict(dtype=3), dict(dtype=0), dict(rows=0), dict(width=0)):
        with pytest.raises(InvalidArgument):
            quantize(name=name, **bad)
    for missing in ("values", "codes", "scales"):
        with pytest.raises(InvalidArgument, match="null operand"):
            quantize(name=name, missing=missing)
    with pytest.raises(InvalidArgument, match="16-byte"):
        quantize(name=name, codes=4104)
    with pytest.raises(LengthError):
        quantize(name=name, width=(1 << 24) + 1)


def test_projection_refusals():
    for bad in (dict(dtype=3), dict(rows=0), dict(inputs=0), dict(outputs=0)):
        with pytest.raises(InvalidArgument):
            project(**bad)
    for missing in ("input", "codes", "scales", "output"):
        with pytest.raises(InvalidArgument, match="null operand"):
            project(missing=missing)
    with pytest.raises(InvalidArgument, match="16-byte"):
        project(codes=4097)
    for large in (dict(rows=(1 << 30) + 1), dict(outputs=(1 << 30) + 1), dict(inputs=(1 << 24) + 1)):
        with pytest.raises(LengthError):
            project(**large)


@pytest.mark.parametrize("field", ["batch", "rows", "query_heads", "kv_heads", "width", "capacity"])
def test_empty_shapes(field):
    empty = shape(**{field: 0})
    with pytest.raises(InvalidArgument):
        attention_workspace_bytes(empty)
    with pytest.raises(InvalidArgument):
        append(empty)
    with pytest.raises(InvalidArgument):
        attend(empty, room=1 << 20)


def test_append_refusals():
    for missing in ("query", "key", "value", "query_out", "lengths", "lengths_out", "positions", "positions_out", "key_codes",
                    "key_scales", "value_codes", "value_scales", "cache"):
        with pytest.raises(InvalidArgument, match="null"):
            append(shape(), missing=missing)
    with pytest.raises(InvalidArgument, match="null shape"):
        append(None)
    with pytest.raises(InvalidArgument, match="even"):
        append(shape(width=63))
    with pytest.raises(InvalidArgument, match="multiple"):
        append(shape(query_heads=7))
    with pytest.raises(InvalidArgument, match="16-byte"):
        append(shape(), held=cache(at="value_codes", address=4100))
    with pytest.raises(InvalidArgument, match="storage"):
        append(shape(), dtype=0)
    for theta in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(InvalidArgument, match="theta"):
            append(shape(), theta=theta)
    for large in (dict(width=258), dict(batch=65536), dict(capacity=(1 << 30) + 1)):
        with pytest.raises(LengthError):
            append(shape(**large))


def test_attention_refusals():
    for missing in ("query", "lengths", "output", "scale", "key_codes", "key_scales", "value_codes", "value_scales", "cache"):
        with pytest.raises(InvalidArgument, match="null"):
            attend(shape(), missing=missing)
    with pytest.raises(InvalidArgument, match="null shape"):
        attend(None, room=0)
    with pytest.raises(InvalidArgument, match="16-byte"):
        attend(shape(), held=cache(at="key_codes", address=4104))
    with pytest.raises(InvalidArgument, match="storage"):
        attend(shape(), dtype=3)
    for large in (dict(width=257), dict(capacity=(1 << 30) + 1), dict(batch=1 << 20, kv_heads=8, query_heads=8)):
        with pytest.raises(LengthError):
            attend(shape(**large), room=1 << 20)
    long = shape(capacity=32768)  # several ranges: a workspace
    room = attention_workspace_bytes(long)
    assert room > 0
    with pytest.raises(InvalidArgument, match="workspace"):
        attend(long, work=0)
    with pytest.raises(InvalidArgument, match="workspace"):
        attend(long, work=4104)
    with pytest.raises(LengthError, match="workspace"):
        attend(long, room=room - 1)
    # A window bounds what a step reads, and so its workspace.
    assert attention_workspace_bytes(long, 256, 4) < room
    assert attention_workspace_bytes(long, 1 << 40) == room


def test_objects_refuse_before_allocating():
    with pytest.raises(InvalidArgument):
        Fp4Cache(None, None, 1, 0, 4, 2, 64)
    with pytest.raises(InvalidArgument):
        Fp4Cache(None, None, 1, 8, 4, 2, 64, dtype="f16")
    with pytest.raises(InvalidArgument):
        Fp4Cache(None, None, 1, 8, 4, 2, 64, window=-1)
    with pytest.raises(InvalidArgument):
        Fp4Weight(None, None, 0, 64)


def test_oracle_rounds_to_the_nearest_code():
    """Borders between neighbouring codes under a scale of one (a 6 fixes it): ties go to the even code."""
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    even = np.array([0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0])
    step = np.array([0.5, 0.5, 0.5, 0.5, 1.0, 1.0, 2.0])
    x = np.concatenate((borders, borders - 1e-6, borders + 1e-6, [6.0, 6.99]))
    codes, scales = ref.quantized(np.concatenate((x, -x[:9]))[None])
    assert scales.tolist() == [[127]]
    got = ref.values(codes, scales, 32)[0]
    want = np.concatenate((even, borders - step / 2, borders + step / 2, [6.0, 6.0]))
    assert np.array_equal(got[:23], want) and np.array_equal(got[23:], -want[:9])


def test_oracle_scales():
    for largest, scale in ((7.0, 128), (6.999, 127), (3.5, 127), (3.499, 126), (0.0, 0), (2.0 ** -140, 0), (3e38, 252),
                           (float("nan"), 255), (float("inf"), 255)):
        x = np.zeros((1, 40))
        x[0, 3] = largest
        codes, scales = ref.quantized(x)
        assert scales[0, 0] == scale and scales[0, 1] == 0 and not codes[0, 1].any()
        assert scale != 255 or not codes.any()
