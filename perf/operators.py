"""Cases of the batch operators over caches that grow and shrink by sequence:
attention of a batch that shares a long prefix, the same attention with the
weight every cached key received, the append of new rows, and the eviction of
the rows that received least.

listed() names the cases, draw() gives more of the same ranges, prepare()
makes what a program holds before the call, run() is one pass (in plain torch
operations, or through the library where `own` is true), exact() the same
result in 64 bits, and work() what a pass has to move and compute.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False

Q_HEADS, KV_HEADS, HEAD, THETA = 32, 8, 128, 1e6
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(kind, batch, rows, prefix, used, dtype="bf16", heads=(Q_HEADS, KV_HEADS, HEAD), **more):
    """`used` is the longest sequence's rows in its own cache, new ones included."""
    return {"kind": kind, "batch": batch, "rows": rows, "prefix": prefix, "used": used, "dtype": dtype,
            "q_heads": heads[0], "kv_heads": heads[1], "width": heads[2], **more}


def listed():
    return [
        # Eight samples of one 192-id prompt, a few tokens in: latency.
        {"name": "shared_decode_8_short", **_case("shared", 8, 1, 192, 24)},
        # The same samples of a long document, some hundred tokens in.
        {"name": "shared_decode_8_long", **_case("shared", 8, 1, 8192, 500)},
        # A serving batch over the longest context a plan holds.
        {"name": "shared_decode_64_longest", **_case("shared", 64, 1, 32768, 1000)},
        # A chunk of 16 new ids per sequence after an odd prefix, FP32 storage.
        {"name": "shared_chunk_16_f32", **_case("shared", 3, 16, 1001, 115, "f32")},
        # Bounded caches in steady decoding: every key's weight is added up.
        {"name": "weighted_decode_8", **_case("weighted", 8, 1, 0, 4607)},
        # FP32 storage, own rows after a shared prefix, odd lengths.
        {"name": "weighted_decode_2_f32", **_case("weighted", 2, 1, 192, 511, "f32")},
        # The last chunk of a long prompt, before the cache is cut to its budget.
        {"name": "weighted_prompt_512", **_case("weighted", 1, 512, 0, 4096)},
        # One row too many: a decode step at the budget.
        {"name": "evict_one", **_case("evict", 8, 1, 0, 2049, budget=2048, sinks=4, recent=256)},
        # Long caches cut to half at once.
        {"name": "evict_half", **_case("evict", 8, 1, 0, 32768, budget=16384, sinks=4, recent=512)},
        # FP32 storage, odd lengths, a sequence that has room left.
        {"name": "evict_odd_f32", **_case("evict", 3, 1, 0, 511, "f32", budget=301, sinks=1, recent=33)},
        # A decode step's new rows of eight sequences at their own positions.
        {"name": "append_8", **_case("append", 8, 1, 0, 2048)},
        # A prompt chunk of two sequences.
        {"name": "append_chunk_512", **_case("append", 2, 512, 0, 1200)},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("shared", "shared", "shared", "weighted", "weighted", "evict", "evict", "append"))
    heads = rng.choice(((32, 8, 128), (32, 8, 128), (16, 2, 64), (8, 8, 128), (12, 4, 80), (8, 1, 256), (40, 8, 96)))
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if kind == "evict":
        used = _log(rng, 40, 32768)
        budget = rng.randint(max(1, used // 4), used)
        recent = rng.randint(0, budget // 2)
        return _bounded(_case(kind, _log(rng, 1, 8), 1, 0, used, dtype, heads, budget=budget,
                              sinks=rng.randint(0, min(8, budget - recent)), recent=recent))
    if kind == "append":
        rows = 1 if rng.random() < 0.5 else _log(rng, 2, 512)
        batch = _log(rng, 1, 64) if rows == 1 else _log(rng, 1, 4)
        return _case(kind, batch, rows, 0, rows + _log(rng, 1, 2048), dtype, heads)
    rows = 1 if rng.random() < 0.6 else _log(rng, 2, 64 if kind == "shared" else 512)
    prefix = _log(rng, 16, 32768) if kind == "shared" or rng.random() < 0.3 else 0
    used = rows + _log(rng, 1, 1000 if kind == "shared" else 8192) - 1
    return _bounded(_case(kind, _log(rng, 1, 64), rows, prefix, used, dtype, heads))


def _bounded(case):
    """The case with fewer sequences, a shorter prefix or fewer new rows, where it costs more than the largest
    listed ones: halved until it does not."""
    limit = 35e9 if case["dtype"] == "bf16" else 9e9
    for field in ("batch", "prefix", "rows", "used"):
        while case[field] > (case["rows"] if field == "used" else 1):
            w = work(case)
            if w["bytes"] <= 300e6 and w["flops"] <= limit:
                return case
            case = {**case, field: case[field] // 2}
    return case


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Rows in use of each sequence's own cache: ragged, never less than the new ones."""
    part = (16, 11, 14, 5, 16, 9, 13, 1)
    return [max(case["rows"], case["used"] * part[b % 8] // 16) for b in range(case["batch"])]


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _keys(g, dtype, *shape):
    """Unit-RMS rows with one in 61 three times as long: the keys that gather attention."""
    k = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
    k[..., ::61, :, :] *= 3.0
    return k.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 6151 + 29)
    t, kind = _TYPES[case["dtype"]], case["kind"]
    batch, rows, used, w = case["batch"], case["rows"], case["used"], case["width"]
    qh, kvh = case["q_heads"], case["kv_heads"]
    capacity = used + 8
    s = {"case": case, "capacity": capacity, "lengths": torch.tensor(_lengths(case), device="cuda"),
         "key": _keys(g, t, batch, capacity, kvh, w), "value": _normal(g, batch, capacity, kvh, w, std=0.8, dtype=t)}
    if kind in ("shared", "weighted"):
        prefix = case["prefix"]
        s["query"] = _normal(g, batch, rows, qh, w, dtype=t)
        s["prefix_key"] = _keys(g, t, prefix, kvh, w)
        s["prefix_value"] = _normal(g, prefix, kvh, w, std=0.8, dtype=t)
        s["scale"] = torch.full((1,), 1.0 / math.sqrt(w), device="cuda")
        s["out"] = torch.zeros_like(s["query"])
        if kind == "weighted":
            s["weights"] = torch.rand(batch, kvh, capacity, generator=g, device="cuda") ** 4
            s["weights_out"] = torch.zeros_like(s["weights"])
        return s
    if kind == "evict":
        # Weights with equal values among them, and positions as earlier evictions leave them, out of order.
        s["weights"] = torch.floor(torch.rand(batch, kvh, capacity, generator=g, device="cuda") ** 4 * 4096) / 64
        order = torch.rand(batch, kvh, capacity, generator=g, device="cuda").argsort(-1)
        s["slots"] = (order * 2 + order % 2).int()
        s["weights_out"], s["slots_out"] = torch.zeros_like(s["weights"]), torch.zeros_like(s["slots"])
        s["lengths_out"] = torch.zeros_like(s["lengths"])
        return s
    # append: the lengths are those before the new rows; positions run ahead of them, rows having been evicted.
    s["lengths"] = s["lengths"] - rows
    s["positions"] = s["lengths"] * 3 + 17
    s["query"] = _normal(g, batch, rows, qh, w, dtype=t)
    s["new_key"], s["new_value"] = _normal(g, batch, rows, kvh, w, dtype=t), _normal(g, batch, rows, kvh, w, std=0.8, dtype=t)
    s["weights"] = torch.rand(batch, kvh, capacity, generator=g, device="cuda")
    s["slots"] = torch.arange(capacity, device="cuda", dtype=torch.int32).expand(batch, kvh, capacity).contiguous()
    s["query_out"] = torch.zeros_like(s["query"])
    s["lengths_out"], s["positions_out"] = torch.zeros_like(s["lengths"]), torch.zeros_like(s["positions"])
    return s


# --------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _own(state)
    if kind in ("shared", "weighted"):
        return _plain_attention(state)
    return _plain_evict(state) if kind == "evict" else _plain_append(state)


def _plain_attention(s):
    c = s["case"]
    b, r, kvh, w, p = c["batch"], c["rows"], c["kv_heads"], c["width"], c["prefix"]
    g, n = c["q_heads"] // kvh, c["used"]
    q = s["query"].float().view(b, r, kvh, g, w)
    k, v = (s[x][:, :n].float().permute(0, 2, 1, 3).contiguous() for x in ("key", "value"))
    pk, pv = (s[x].float().permute(1, 0, 2).contiguous() for x in ("prefix_key", "prefix_value"))
    # The prefix: all queries of a KV head against one set of keys.
    shared = q.permute(2, 0, 1, 3, 4).reshape(kvh, b * r * g, w)
    before = (shared @ pk.transpose(1, 2)).view(kvh, b, r, g, p).permute(1, 0, 2, 3, 4).reshape(b, kvh, r * g, p)
    mine = q.permute(0, 2, 1, 3, 4).reshape(b, kvh, r * g, w) @ k.transpose(2, 3)
    # New row i of a sequence sees its own rows up to itself.
    last = s["lengths"][:, None] - r + torch.arange(r, device="cuda")
    hidden = (torch.arange(n, device="cuda") > last[..., None]).repeat_interleave(g, 1)[:, None]
    scores = torch.cat((before, mine.masked_fill(hidden, -math.inf)), -1) * s["scale"]
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    e = e / e.sum(-1, keepdim=True)
    old = e[..., :p].reshape(b, kvh, r, g, p).permute(1, 0, 2, 3, 4).reshape(kvh, b * r * g, p) @ pv
    out = old.view(kvh, b, r, g, w).permute(1, 2, 0, 3, 4) + (e[..., p:] @ v).view(b, kvh, r, g, w).permute(0, 2, 1, 3, 4)
    out = out.reshape(b, r, c["q_heads"], w).to(s["query"].dtype)
    if c["kind"] == "shared":
        return {"out": out}
    total = s["weights"].clone()
    total[..., :n] += e[..., p:].sum(2)
    used = torch.arange(s["capacity"], device="cuda") < s["lengths"][:, None, None]
    return {"out": out, "weights": torch.where(used, total, torch.zeros_like(total))}


def _plain_evict(s):
    c = s["case"]
    budget, n = c["budget"], s["lengths"]
    slot = torch.arange(s["capacity"], device="cuda")
    used = (slot < n[:, None, None]).expand_as(s["weights"])
    at = s["slots"].long()
    newest = at.masked_fill(~used, -1).amax(-1, keepdim=True)
    safe = (at < c["sinks"]) | (at + c["recent"] > newest)
    # Order of keeping: in use, protected, larger weight, lower slot.
    order = torch.argsort(s["weights"], dim=-1, descending=True, stable=True)
    grade = used.int() + (used & safe).int()
    order = order.gather(-1, torch.argsort(grade.gather(-1, order), dim=-1, descending=True, stable=True))
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order))
    kept = used & (rank < budget)
    left = n.clamp(max=budget)
    inside = slot < left[:, None, None]
    # The j-th slot below the new length that is not kept takes the j-th kept row above it.
    hole, filler = inside & ~kept, ~inside & kept
    place = torch.where(filler, filler.cumsum(-1) - 1, torch.full_like(order, s["capacity"]))
    listed_ = torch.zeros(*order.shape[:2], s["capacity"] + 1, dtype=torch.long, device="cuda")
    listed_.scatter_(-1, place, slot.expand_as(order))
    source = torch.where(hole, listed_.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), slot)[..., :budget]
    rows = source.permute(0, 2, 1)[..., None].expand(-1, -1, -1, c["width"])
    for x in ("key", "value"):
        s[x][:, :budget] = s[x].gather(1, rows)
    for x in ("weights", "slots"):
        s[x + "_out"][..., :budget] = torch.where(inside[..., :budget], s[x].gather(-1, source), torch.zeros_like(s[x][..., :budget]))
    return {"key": s["key"], "value": s["value"], "weights": s["weights_out"], "slots": s["slots_out"], "lengths": left}


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
        return torch.cat((lo * cosine - hi * sine, hi * cosine + lo * sine), -1).to(x.dtype)

    row = s["lengths"][:, None] + at
    sequence = torch.arange(b, device="cuda")[:, None].expand(b, r)
    s["key"][sequence, row] = turned(s["new_key"])
    s["value"][sequence, row] = s["new_value"]
    s["weights"].transpose(1, 2)[sequence, row] = 0.0
    s["slots"].transpose(1, 2)[sequence, row] = (s["positions"][:, None] + at).int()[..., None].expand(b, r, c["kv_heads"])
    return {"query": turned(s["query"]), "key": s["key"], "value": s["value"], "weights": s["weights"],
            "slots": s["slots"], "lengths": s["lengths"] + r, "positions": s["positions"] + r}


def _call(s):
    """The library's function, its arguments and what it fills, made once as a program does."""
    from dolittle_amd import _lib
    from dolittle_amd.batch import BatchShape, workspace_bytes
    c, kind = s["case"], s["case"]["kind"]
    shape = BatchShape(c["batch"], c["rows"], c["q_heads"], c["kv_heads"], c["width"], s["capacity"])
    code = 1 if c["dtype"] == "bf16" else 2
    p = {n: C.c_void_p(t.data_ptr()) for n, t in s.items() if isinstance(t, torch.Tensor)}
    head = (_queue().handle, code, C.byref(shape))
    if kind in ("shared", "weighted"):
        name = "dl_attention_" + kind
        room = workspace_bytes(name, shape, c["prefix"])
        args = (p["query"], p["prefix_key"] if c["prefix"] else None, p["prefix_value"] if c["prefix"] else None,
                c["prefix"], p["key"], p["value"], p["lengths"])
        if kind == "weighted":
            args += p["weights"], p["weights_out"]
        args += p["out"], p["scale"]
        filled = {"out": s["out"], "weights": s["weights_out"]} if kind == "weighted" else {"out": s["out"]}
    elif kind == "evict":
        name = "dl_cache_evict"
        room = workspace_bytes(name, shape, c["budget"])
        args = (p["key"], p["value"], p["lengths"], p["lengths_out"], p["slots"], p["slots_out"], p["weights"],
                p["weights_out"], c["budget"], c["sinks"], c["recent"])
        filled = {"key": s["key"], "value": s["value"], "weights": s["weights_out"], "slots": s["slots_out"],
                  "lengths": s["lengths_out"]}
    else:
        name, room = "dl_cache_append", 0
        args = (p["query"], p["new_key"], p["new_value"], p["query_out"], p["key"], p["value"], p["lengths"],
                p["lengths_out"], p["positions"], p["positions_out"], p["slots"], p["weights"], C.c_double(THETA))
        filled = {"query": s["query_out"], "key": s["key"], "value": s["value"], "weights": s["weights"],
                  "slots": s["slots"], "lengths": s["lengths_out"], "positions": s["positions_out"]}
    if room:
        s["workspace"] = torch.empty(room, dtype=torch.uint8, device="cuda")
        args += C.c_void_p(s["workspace"].data_ptr()), C.c_uint64(room)
    torch.cuda.synchronize()
    return getattr(_lib.load(), name), head + args, filled, _lib.check, shape


def _own(s):
    if "call" not in s:
        s["call"] = _call(s)
    function, args, filled, check, _ = s["call"]
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
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    b, r, w, kvh, qh = (case[x] for x in ("batch", "rows", "width", "kv_heads", "q_heads"))
    lengths = _lengths(case)
    row = kvh * w * size
    if case["kind"] == "append":
        return {"bytes": b * r * (2 * qh * w * size + 4 * row + 8 * kvh) + 32 * b, "flops": 3 * b * r * (qh + kvh) * w}
    if case["kind"] == "evict":
        # Weights and positions of every row, those kept again, and the expected number of rows that move.
        moved = sum((n - case["budget"]) * case["budget"] / n for n in lengths if n > case["budget"])
        kept = sum(min(n, case["budget"]) for n in lengths)
        return {"bytes": int(8 * kvh * (sum(lengths) + kept) + 4 * moved * row), "flops": 4 * kvh * sum(lengths)}
    pairs = sum(r * (case["prefix"] + n - r) + r * (r + 1) // 2 for n in lengths)
    moved = 2 * (case["prefix"] + sum(lengths)) * row + 2 * b * r * qh * w * size
    if case["kind"] == "weighted":
        moved += 8 * kvh * sum(lengths)
    return {"bytes": moved, "flops": 4 * pairs * qh * w}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"shared": _exact_attention, "weighted": _exact_attention, "evict": _exact_evict,
            "append": _exact_append}[case["kind"]](case, s)


def _exact_attention(case, s):
    """One sequence and one KV head at a time, in 64 bits."""
    r, kvh, p = case["rows"], case["kv_heads"], case["prefix"]
    g = case["q_heads"] // kvh
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    weights = torch.zeros(case["batch"], kvh, s["capacity"], dtype=torch.float64, device="cuda")
    factor = float(s["scale"])
    for h in range(kvh):
        pk, pv = s["prefix_key"][:, h].double(), s["prefix_value"][:, h].double()
        for b, n in enumerate(_lengths(case)):
            k = torch.cat((pk, s["key"][b, :n, h].double()))
            v = torch.cat((pv, s["value"][b, :n, h].double()))
            q = s["query"][b, :, h * g:(h + 1) * g].double().reshape(r * g, -1)
            late = torch.arange(p + n, device="cuda")[None] > p + n - r + torch.arange(r, device="cuda")[:, None]
            score = (q @ k.t().contiguous() * factor).masked_fill(late.repeat_interleave(g, 0), -math.inf)
            share = torch.softmax(score, -1)
            out[b, :, h * g:(h + 1) * g] = (share @ v).view(r, g, -1)
            weights[b, h, :n] = s["weights"][b, h, :n].double() + share[:, p:].sum(0) if "weights" in s else 0.0
    return {"out": out} if case["kind"] == "shared" else {"out": out, "weights": weights}


def _exact_evict(case, s):
    """The kept rows by sorting on the host; the caches' values are only moved."""
    budget, lengths = case["budget"], _lengths(case)
    weights, slots = s["weights"].cpu().numpy(), s["slots"].cpu().numpy()
    key, value = s["key"].double(), s["value"].double()
    got = np.zeros(weights.shape)
    for b, n in enumerate(lengths):
        left = min(n, budget)
        for h in range(case["kv_heads"]):
            wt, at = weights[b, h, :n], slots[b, h, :n].astype(np.int64)
            source = np.arange(left)
            if n > budget:
                safe = (at < case["sinks"]) | (at > at.max() - case["recent"])
                kept = np.zeros(n, bool)
                kept[np.lexsort((np.arange(n), -wt, ~safe))[:budget]] = True
                source[~kept[:budget]] = budget + np.flatnonzero(kept[budget:])
            got[b, h, :left] = wt[source]
            source = torch.from_numpy(source).cuda()
            key[b, :left, h], value[b, :left, h] = key[b, source, h], value[b, source, h]
    return {"key": key, "value": value, "weights": torch.from_numpy(got), "slots": None, "lengths": None}


def _exact_append(case, s):
    r, half = case["rows"], case["width"] // 2
    exponent = (2 * np.arange(half)).astype(np.float32) / np.float32(case["width"])
    frequency = (1.0 / THETA ** exponent.astype(np.float64)).astype(np.float32)
    first, start = s["positions"].cpu().numpy(), s["lengths"].cpu().numpy()
    key, value, query = s["key"].double(), s["value"].double(), s["query"].double()
    weights = s["weights"].double()
    for b in range(case["batch"]):
        angle = torch.from_numpy((first[b] + np.arange(r)).astype(np.float32)[:, None] * frequency).cuda().double()
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        rows = slice(int(start[b]), int(start[b]) + r)
        for x, into in ((s["query"][b].double(), query[b]), (s["new_key"][b].double(), key[b, rows])):
            z = torch.complex(x[..., :half], x[..., half:]) * turn
            into.copy_(torch.cat((z.real, z.imag), -1))
        value[b, rows] = s["new_value"][b].double()
        weights[b, :, rows] = 0.0
    return {"query": query, "key": key, "value": value, "weights": weights, "slots": None, "lengths": None,
            "positions": None}
