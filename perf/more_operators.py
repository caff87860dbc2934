"""Cases of the operators over 4-bit storage: rows quantised to 4 bits with a
scale for every 32 values, the projection by such weights, the append of
rotated keys and values to a cache held in 4 bits, and the attention over such
a cache, with or without a sliding window and first rows that stay visible.

listed() names the cases, draw() gives more of the same ranges, prepare()
makes what a program holds before the call, run() is one pass (in plain torch
operations, or through the library where `own` is true), exact() the same
result in 64 bits, and work() what a pass has to move and compute.

A row of `width` values is ceil(width / 32) groups; a group is 16 bytes, the
lower half of a byte the earlier value, and one scale byte s.  A value's four
bits are its sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6; it stands for that
times 2^(s - 127).  Weights are [outputs][groups], caches
[batch][kv_heads][capacity][groups].
"""
from __future__ import annotations

import ctypes as C
import math

import torch

own = False

HIDDEN, KV_WIDTH, QKV_WIDTH, FFN, VOCABULARY = 4096, 1024, 6144, 12288, 151936
HEADS, THETA = (32, 8, 128), 1e6
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _project(rows, inputs, outputs, dtype="bf16"):
    return {"kind": "project", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype}


def _cached(kind, batch, rows, used, dtype="bf16", heads=HEADS, **more):
    """`used` is the longest sequence's rows in its cache, new ones included."""
    return {"kind": kind, "batch": batch, "rows": rows, "used": used, "dtype": dtype, "q_heads": heads[0],
            "kv_heads": heads[1], "width": heads[2], **more}


def _attend(batch, rows, used, dtype="bf16", heads=HEADS, window=0, sinks=0):
    return _cached("attend", batch, rows, used, dtype, heads, window=window, sinks=sinks)


def _quantize(rows, width, dtype="bf16"):
    return {"kind": "quantize", "rows": rows, "width": width, "dtype": dtype}


def listed():
    return [
        # The key projection of one decode step: latency.
        {"name": "project_key_1", **_project(1, HIDDEN, KV_WIDTH)},
        # The vocabulary's logits of eight sequences: the largest weight there is.
        {"name": "project_head_8", **_project(8, HIDDEN, VOCABULARY)},
        # Query, key and value of a prompt chunk.
        {"name": "project_chunk_512", **_project(512, HIDDEN, QKV_WIDTH)},
        # Three rows through the down projection in FP32 storage, an odd number of outputs.
        {"name": "project_down_3_f32", **_project(3, FFN, 4095, "f32")},
        # A decode step early in three answers, FP32 storage, head rows with a short last group.
        {"name": "attend_3_short_f32", **_attend(3, 1, 201, "f32", (12, 4, 80))},
        # A serving batch over long contexts.
        {"name": "attend_64_longest", **_attend(64, 1, 32768)},
        # Decoding behind long contexts with the last 1024 rows and the first four in sight.
        {"name": "attend_8_window", **_attend(8, 1, 32768, window=1024, sinks=4)},
        # An odd prompt chunk under a window that ends inside it.
        {"name": "attend_chunk_window", **_attend(1, 1000, 5001, window=511, sinks=4)},
        # A decode step's new rows of eight sequences at their own positions.
        {"name": "append_8", **_cached("append", 8, 1, 200)},
        # A prompt chunk of two sequences, FP32 storage.
        {"name": "append_chunk_512_f32", **_cached("append", 2, 512, 1200, "f32")},
        # The gate projection's weights, once when a model is loaded.
        {"name": "quantize_gate", **_quantize(FFN, HIDDEN)},
        # A few FP32 rows with a short last group.
        {"name": "quantize_rows_f32", **_quantize(37, 1000, "f32")},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("project", "project", "project", "attend", "attend", "attend", "append", "quantize"))
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if kind == "project":
        rows = _log(rng, 1, 16) if rng.random() < 0.6 else _log(rng, 17, 512)
        inputs = rng.choice((HIDDEN, FFN, KV_WIDTH)) if rng.random() < 0.5 else _log(rng, 48, FFN)
        return _bounded(_project(rows, inputs, _log(rng, 64, VOCABULARY), dtype), ("outputs", "rows"))
    if kind == "quantize":
        return _bounded(_quantize(_log(rng, 8, FFN), _log(rng, 48, HIDDEN), dtype), ("rows",))
    heads = rng.choice((HEADS, HEADS, (16, 2, 64), (8, 8, 128), (12, 4, 80), (8, 1, 256), (40, 8, 96)))
    if kind == "append":
        rows = 1 if rng.random() < 0.5 else _log(rng, 2, 512)
        batch = _log(rng, 1, 16) if rows == 1 else _log(rng, 1, 4)
        return _cached(kind, batch, rows, rows + _log(rng, 1, 700), dtype, heads)
    rows = 1 if rng.random() < 0.6 else _log(rng, 2, 1000)
    window = 0 if rng.random() < 0.5 else _log(rng, 16, 4096)
    case = _attend(_log(rng, 1, 64), rows, rows + _log(rng, 1, 32768) - 1, dtype, heads, window,
                   rng.randint(0, 8) if window else 0)
    return _bounded(case, ("batch", "used", "rows"))


def _bounded(case, fields):
    """The case halved, field by field, until it costs no more than the largest listed ones."""
    limit = 3e10 if case["dtype"] == "bf16" else 1e10
    if case["kind"] == "attend":
        limit = 4e10 if case["dtype"] == "bf16" else 1e10
    for field in fields:
        while case[field] > (case["rows"] if field == "used" else 1):
            w = work(case)
            held = case["batch"] * case["used"] * case["kv_heads"] * case["width"] if case["kind"] == "attend" else 0
            if w["bytes"] <= 350e6 * (4 if case["kind"] == "attend" else 1) and w["flops"] <= limit and held <= 1 << 31:
                return case
            case = {**case, field: case[field] // 2}
            if "used" in case:
                case["used"] = max(case["used"], case["rows"])
    return case


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Rows in use of each sequence's cache: ragged, never less than the new ones."""
    part = (16, 11, 14, 5, 16, 9, 13, 1)
    return [max(case["rows"], case["used"] * part[b % 8] // 16) for b in range(case["batch"])]


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _held_weights(g, outputs, inputs):
    """Codes and scales of normal weights whose outputs have the inputs' size; some rows are larger."""
    codes, scales = [], []
    for first in range(0, outputs, 16384):
        x = _normal(g, min(16384, outputs - first), inputs, std=inputs ** -0.5, dtype=torch.float32)
        x[::61] *= 3.0
        for to, part in zip((codes, scales), _packed(x)):
            to.append(part)
    return torch.cat(codes), torch.cat(scales)


def _held_rows(g, batch, kv_heads, capacity, width, std, tall=False):
    """Codes and scales of cached rows; with `tall` one row in 61 is three times as long: keys that gather attention."""
    codes, scales = [], []
    for _ in range(batch):
        x = _normal(g, kv_heads, capacity, width, std=std, dtype=torch.float32)
        if tall:
            x[:, ::61] *= 3.0
        for to, part in zip((codes, scales), _packed(x)):
            to.append(part)
    return torch.stack(codes), torch.stack(scales)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 43)
    t, kind = _TYPES[case["dtype"]], case["kind"]
    s = {"case": case}
    if kind == "project":
        s["input"] = _normal(g, case["rows"], case["inputs"], dtype=t)
        s["codes"], s["scales"] = _held_weights(g, case["outputs"], case["inputs"])
        s["out"] = torch.zeros(case["rows"], case["outputs"], device="cuda", dtype=t)
        return s
    if kind == "quantize":
        s["input"] = _normal(g, case["rows"], case["width"], std=case["width"] ** -0.5, dtype=t)
        groups = -(-case["width"] // 32)
        s["codes"] = torch.zeros(case["rows"], groups, 16, device="cuda", dtype=torch.uint8)
        s["scales"] = torch.zeros(case["rows"], groups, device="cuda", dtype=torch.uint8)
        s["values"] = torch.zeros_like(s["input"])
        return s
    batch, rows, used, w = case["batch"], case["rows"], case["used"], case["width"]
    qh, kvh = case["q_heads"], case["kv_heads"]
    s["capacity"] = capacity = used + 8
    s["lengths"] = torch.tensor(_lengths(case), device="cuda")
    s["key_codes"], s["key_scales"] = _held_rows(g, batch, kvh, capacity, w, 1.0, True)
    s["value_codes"], s["value_scales"] = _held_rows(g, batch, kvh, capacity, w, 0.8)
    s["query"] = _normal(g, batch, rows, qh, w, dtype=t)
    s["out"] = torch.zeros_like(s["query"])
    if kind == "attend":
        s["scale"] = torch.full((1,), 1.0 / math.sqrt(w), device="cuda")
        return s
    # append: the lengths are those before the new rows; the positions run ahead of them, behind a dropped beginning.
    s["lengths"] = s["lengths"] - rows
    s["positions"] = s["lengths"] * 3 + 17
    s["new_key"], s["new_value"] = _normal(g, batch, rows, kvh, w, dtype=t), _normal(g, batch, rows, kvh, w, std=0.8, dtype=t)
    s["lengths_out"], s["positions_out"] = torch.zeros_like(s["lengths"]), torch.zeros_like(s["positions"])
    s["keys"] = torch.zeros(batch, kvh, capacity, w, device="cuda", dtype=torch.bfloat16)
    s["values"] = torch.zeros_like(s["keys"])
    return s


# -------------------------------------------------------- the 4-bit format
_BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)  # between neighbouring values; ties go to the even code
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _packed(x):
    """Codes [..., groups, 16] and scales [..., groups] of FP32 rows.  The scale is the power of two under which the
    group's largest value lies below 7 and not below 3.5 (no value then lies past 6 by more than half a step)."""
    groups = -(-x.shape[-1] // 32)
    x = torch.nn.functional.pad(x, (0, groups * 32 - x.shape[-1])).reshape(*x.shape[:-1], groups, 32)
    largest = x.abs().amax(-1)
    scales = (((largest.view(torch.int32) + 0x200000) >> 23) - 2).clamp(0, 252)
    factor = ((254 - scales) << 23).view(torch.float32)
    y = (x * factor[..., None]).abs()
    code = torch.signbit(x).to(torch.uint8) * 8
    for i, border in enumerate(_BORDERS):
        code += (y >= border if i % 2 else y > border)
    finite = torch.isfinite(largest)
    code *= finite[..., None]
    return code[..., ::2] | (code[..., 1::2] << 4), torch.where(finite, scales, 255).to(torch.uint8)


def _values(codes, scales, width):
    """The FP32 values that codes and scales stand for."""
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), device=codes.device)
    byte = torch.arange(256, device=codes.device)
    pairs = torch.stack((grid[byte % 16], grid[byte // 16]), -1)
    bits = scales.int() << 23
    bits = torch.where(scales == 0, 0x00400000, torch.where(scales == 255, 0x7fc00000, bits))
    x = pairs[codes.int()].flatten(-2) * bits.view(torch.float32)[..., None]
    return x.flatten(-2)[..., :width]


# --------------------------------------------------------------------- run
def run(state):
    if own:
        return _own(state)
    return {"project": _plain_project, "attend": _plain_attend, "append": _plain_append,
            "quantize": _plain_quantize}[state["case"]["kind"]](state)


def _plain_project(s):
    w = _values(s["codes"], s["scales"], s["case"]["inputs"])
    return {"out": (s["input"].float() @ w.t()).to(s["input"].dtype)}


def _plain_quantize(s):
    codes, scales = _packed(s["input"].float())
    return {"values": _values(codes, scales, s["case"]["width"]).to(s["input"].dtype)}


def _plain_attend(s):
    c = s["case"]
    b, r, kvh, w, n, window, sinks = (c[x] for x in ("batch", "rows", "kv_heads", "width", "used", "window", "sinks"))
    g = c["q_heads"] // kvh
    # New row i of a sequence is at its own slot; it sees the slots up to that one, the last `window` of them or the
    # first `sinks`.  Under a window only the rows that some new row sees are taken.
    at = (s["lengths"][:, None] - r + torch.arange(r, device="cuda"))[..., None]
    slot = torch.arange(n, device="cuda").expand(b, n)
    if window and sinks + window + r - 1 < n:
        first = (s["lengths"] - r + 1 - window).clamp(min=sinks)[:, None]
        slot = torch.cat((slot[:, :sinks], first + torch.arange(window + r - 1, device="cuda")), 1)
    seen = slot[:, None] <= at
    if window:
        seen &= (slot[:, None] > at - window) | (slot[:, None] < sinks)

    def held(name):
        codes, scales = s[name + "_codes"][:, :, :n], s[name + "_scales"][:, :, :n]
        if slot.shape[1] < n:
            row = torch.arange(b, device="cuda")[:, None], slot.clamp(max=n - 1)
            codes, scales = codes.transpose(1, 2)[row].transpose(1, 2), scales.transpose(1, 2)[row].transpose(1, 2)
        return _values(codes, scales, w)

    q = s["query"].float().view(b, r, kvh, g, w).permute(0, 2, 1, 3, 4).reshape(b, kvh, r * g, w)
    scores = (q @ held("key").transpose(2, 3)) * s["scale"]
    scores = scores.masked_fill_(~seen.repeat_interleave(g, 1)[:, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    out = e @ held("value")
    return {"out": out.view(b, kvh, r, g, w).permute(0, 2, 1, 3, 4).reshape(b, r, c["q_heads"], w).to(s["query"].dtype)}


def _angles(positions, w):
    """FP32 angles of the rotation: the FP32 position times an FP32 frequency."""
    exponent = (torch.arange(w // 2, device="cuda") * 2).float() / float(w)
    frequency = (1.0 / THETA ** exponent.double()).float()
    return positions.float()[..., None] * frequency


def _plain_append(s):
    c = s["case"]
    b, r, w = c["batch"], c["rows"], c["width"]
    at = torch.arange(r, device="cuda")
    angle = _angles(s["positions"][:, None] + at, w).double()[:, :, None]
    cosine, sine = torch.cos(angle).float(), torch.sin(angle).float()

    def turned(x):
        lo, hi = x.float()[..., :w // 2], x.float()[..., w // 2:]
        return torch.cat((lo * cosine - hi * sine, hi * cosine + lo * sine), -1)

    row = s["lengths"][:, None] + at
    sequence = torch.arange(b, device="cuda")[:, None].expand(b, r)
    for x, name in ((turned(s["new_key"]), "key"), (s["new_value"].float(), "value")):
        codes, scales = _packed(x)
        s[name + "_codes"].transpose(1, 2)[sequence, row] = codes
        s[name + "_scales"].transpose(1, 2)[sequence, row] = scales
    return {"query": turned(s["query"]).to(s["query"].dtype), "lengths": s["lengths"] + r, "positions": s["positions"] + r,
            "key": _values(s["key_codes"], s["key_scales"], w).bfloat16(),
            "value": _values(s["value_codes"], s["value_scales"], w).bfloat16()}


def _calls(s):
    """The library's functions with their arguments, and what they fill, made once as a program does."""
    from dolittle_amd import _lib
    from dolittle_amd.batch import BatchShape
    from dolittle_amd.fp4 import CacheAddresses, attention_workspace_bytes
    c, kind, queue = s["case"], s["case"]["kind"], _queue().handle
    code = 1 if c["dtype"] == "bf16" else 2
    p = {n: C.c_void_p(t.data_ptr()) for n, t in s.items() if isinstance(t, torch.Tensor)}
    if kind == "project":
        calls = [("dl_projection_fp4", (queue, code, p["input"], p["codes"], p["scales"], p["out"], c["rows"], c["inputs"],
                                        c["outputs"], None))]
        filled, held = {"out": s["out"]}, None
    elif kind == "quantize":
        calls = [("dl_fp4_quantize", (queue, code, p["input"], p["codes"], p["scales"], c["rows"], c["width"])),
                 ("dl_fp4_values", (queue, code, p["codes"], p["scales"], p["values"], c["rows"], c["width"]))]
        filled, held = {"values": s["values"]}, None
    else:
        shape = BatchShape(c["batch"], c["rows"], c["q_heads"], c["kv_heads"], c["width"], s["capacity"])
        cache = CacheAddresses(p["key_codes"], p["key_scales"], p["value_codes"], p["value_scales"])
        held = shape, cache
        if kind == "attend":
            room = attention_workspace_bytes(shape, c["window"], c["sinks"])
            s["workspace"] = torch.empty(max(room, 16), dtype=torch.uint8, device="cuda")
            calls = [("dl_attention_fp4", (queue, code, C.byref(shape), p["query"], C.byref(cache), p["lengths"], c["window"],
                                           c["sinks"], p["out"], p["scale"], C.c_void_p(s["workspace"].data_ptr()),
                                           C.c_uint64(room)))]
            filled = {"out": s["out"]}
        else:
            rows = c["batch"] * c["kv_heads"] * s["capacity"]
            calls = [("dl_cache_append_fp4", (queue, code, C.byref(shape), p["query"], p["new_key"], p["new_value"], p["out"],
                                              C.byref(cache), p["lengths"], p["lengths_out"], p["positions"],
                                              p["positions_out"], C.c_double(THETA))),
                     ("dl_fp4_values", (queue, 1, p["key_codes"], p["key_scales"], p["keys"], rows, c["width"])),
                     ("dl_fp4_values", (queue, 1, p["value_codes"], p["value_scales"], p["values"], rows, c["width"]))]
            filled = {"query": s["out"], "lengths": s["lengths_out"], "positions": s["positions_out"], "key": s["keys"],
                      "value": s["values"]}
    torch.cuda.synchronize()
    library = _lib.load()
    return [(getattr(library, name), args) for name, args in calls], filled, _lib.check, held


def _own(s):
    if "calls" not in s:
        s["calls"] = _calls(s)
    calls, filled, check, _ = s["calls"]
    for function, args in calls:
        check(function(*args))
    return filled


_open = {}


def _queue():
    if not _open:
        from dolittle_amd import Device
        _open["device"] = Device(0)
        _open["queue"] = _open["device"].create_queue()
    return _open["queue"]


# -------------------------------------------------------------------- work
def _row_bytes(width):
    """Codes and scales of one row; a last group counts with its values."""
    return (width + 1) // 2 + -(-width // 32)


def _seen(case, n):
    """(rows that any new row of a sequence of n sees, pairs of a new row and a row that it sees)."""
    r, window, sinks = case["rows"], case["window"], case["sinks"]
    if not window:
        return n, r * (n - r) + r * (r + 1) // 2
    low = max(0, n - r + 1 - window)
    pairs = sum(min(at + 1, window) + min(sinks, max(0, at + 1 - window)) for at in range(n - r, n))
    return n - low + min(sinks, low), pairs


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "project":
        r, i, o = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": o * _row_bytes(i) + r * (i + o) * size, "flops": 2 * r * i * o}
    if case["kind"] == "quantize":
        r, w = case["rows"], case["width"]
        return {"bytes": r * (2 * w * size + _row_bytes(w)), "flops": 4 * r * w}
    b, r, w, kvh, qh = (case[x] for x in ("batch", "rows", "width", "kv_heads", "q_heads"))
    if case["kind"] == "append":
        held = b * kvh * (case["used"] + 8)
        return {"bytes": b * r * (2 * qh + 2 * kvh) * w * size + 32 * b + 2 * held * (_row_bytes(w) + 2 * w),
                "flops": 3 * b * r * (qh + kvh) * w + 2 * held * w}
    seen = [_seen(case, n) for n in _lengths(case)]
    return {"bytes": 2 * sum(k for k, _ in seen) * kvh * _row_bytes(w) + 2 * b * r * qh * w * size,
            "flops": 4 * sum(p for _, p in seen) * qh * w}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"project": _exact_project, "attend": _exact_attend, "append": _exact_append,
            "quantize": _exact_quantize}[case["kind"]](case, s)


def _decoded(codes, scales, width):
    """The values in 64 bits, bit by bit: sign, two of exponent, one of fraction."""
    nibble = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    exponent, fraction = (nibble >> 1) & 3, (nibble & 1).double()
    size = torch.where(exponent == 0, fraction / 2, (1 + fraction / 2) * torch.exp2((exponent - 1).double()))
    size = torch.where(nibble >= 8, -size, size) * torch.ldexp(torch.ones((), dtype=torch.float64, device=codes.device),
                                                                scales.int() - 127)[..., None]
    return size.flatten(-2)[..., :width]


def _rounded(x):
    """64-bit rows rounded to the values that 4 bits and the group's scale can stand for."""
    width, groups = x.shape[-1], -(-x.shape[-1] // 32)
    x = torch.nn.functional.pad(x, (0, groups * 32 - width)).unflatten(-1, (groups, 32))
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    scale = torch.ldexp(torch.ones_like(mantissa), exponent - 3 + (mantissa >= 0.875).int())
    y = (x / scale).abs()
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0)).double()
    y = torch.minimum(torch.round(y / step) * step, torch.full_like(y, 6.0))
    return (torch.copysign(y, x) * scale).flatten(-2)[..., :width]


def _exact_project(case, s):
    x = s["input"].double()
    parts = [x @ _decoded(s["codes"][o:o + 8192], s["scales"][o:o + 8192], case["inputs"]).t()
             for o in range(0, case["outputs"], 8192)]
    return {"out": torch.cat(parts, -1)}


def _exact_quantize(case, s):
    return {"values": _rounded(s["input"].double())}


def _exact_attend(case, s):
    """One sequence and one KV head at a time, in 64 bits."""
    r, kvh, w, window, sinks = (case[x] for x in ("rows", "kv_heads", "width", "window", "sinks"))
    g = case["q_heads"] // kvh
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    factor = float(s["scale"])
    for b, n in enumerate(_lengths(case)):
        slot, at = torch.arange(n, device="cuda"), n - r + torch.arange(r, device="cuda")[:, None]
        hidden = slot > at
        if window:
            hidden |= (at - slot >= window) & (slot >= sinks)
        hidden = hidden.repeat_interleave(g, 0)
        for h in range(kvh):
            k = _decoded(s["key_codes"][b, h, :n], s["key_scales"][b, h, :n], w)
            v = _decoded(s["value_codes"][b, h, :n], s["value_scales"][b, h, :n], w)
            q = s["query"][b, :, h * g:(h + 1) * g].double().reshape(r * g, w)
            score = (q @ k.t() * factor).masked_fill(hidden, -math.inf)
            out[b, :, h * g:(h + 1) * g] = (torch.softmax(score, -1) @ v).view(r, g, w)
    return {"out": out}


def _exact_append(case, s):
    r, w = case["rows"], case["width"]
    half = w // 2
    place = torch.arange(half, dtype=torch.float32, device="cuda")
    frequency = (1.0 / torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"), (2 * place / w).double())).float()
    key, value = (_decoded(s[x + "_codes"], s[x + "_scales"], w) for x in ("key", "value"))
    query = torch.empty(s["query"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        first, start = int(s["positions"][b]), int(s["lengths"][b])
        angle = (torch.arange(first, first + r, device="cuda").float()[:, None] * frequency).double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]

        def turned(x):
            z = torch.complex(x[..., :half], x[..., half:]) * turn
            return torch.cat((z.real, z.imag), -1)

        query[b] = turned(s["query"][b].double())
        key[b, :, start:start + r] = _rounded(turned(s["new_key"][b].double())).transpose(0, 1)
        value[b, :, start:start + r] = _rounded(s["new_value"][b].double()).transpose(0, 1)
    return {"query": query, "key": key, "value": value, "lengths": None, "positions": None}
