"""64-bit definitions of the operations over 4-bit storage, written from their
formulas, and the error bounds of the tests.

Bounds.  u is half a step of the storage type (BF16 2^-8, FP32 2^-24), all
relative.  The values that codes and scales stand for are exact in BF16, and so
are the products of the matrix cores.  A sum of n FP32 terms in any order is off
by at most n 2^-24 of the sum of their magnitudes; FP32 inputs run as three exact
parts, three times as many terms.  Attention as in batch_reference: a score is off by its sum's
bound, an exponential by that, by the exponent's two roundings (2^-23 of the
difference to the maximum) and by two steps of the hardware's exp2; BF16 storage
rounds each exponential once more (u) and every result once (u)."""
import numpy as np

HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}
PARTS = {"bf16": 1, "f32": 3}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def groups_of(width):
    return -(-width // 32)


def values(codes, scales, width):
    """codes [..., G, 16], scales [..., G] -> float64 [..., width]."""
    nibbles = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], 32)
    x = np.where(nibbles >= 8, -1.0, 1.0) * GRID[nibbles & 7]
    factor = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (x * factor[..., None]).reshape(*codes.shape[:-2], -1)[..., :width]


def quantized(x):
    """float64 rows [..., width] (values of FP32) -> codes [..., G, 16], scales [..., G].  The nearest value by
    search; of two that are as near, the even code."""
    width, groups = x.shape[-1], groups_of(x.shape[-1])
    x = np.concatenate((x, np.zeros((*x.shape[:-1], groups * 32 - width))), -1).reshape(*x.shape[:-1], groups, 32)
    finite = np.isfinite(x).all(-1)
    clean = np.where(finite[..., None], x, 0.0)
    largest = np.abs(clean).max(-1)
    scales = np.zeros(largest.shape, np.int64)
    for s in range(252, -1, -1):  # the smallest scale under which the largest magnitude is below 7
        scales[largest < np.ldexp(7.0, s - 127)] = s
    scales[largest >= np.ldexp(7.0, 252 - 127)] = 252
    y = np.abs(clean) / np.ldexp(1.0, scales - 127)[..., None]
    far = np.abs(y[..., None] - GRID)
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])  # even codes first: argmin takes the first of equals
    code = order[np.argmin(far[..., order], -1)] | (np.signbit(clean).astype(np.int64) << 3)
    code = np.where(finite[..., None], code, 0).astype(np.uint8)
    return code[..., ::2] | (code[..., 1::2] << 4), np.where(finite, scales, 255).astype(np.uint8)


def projection(x, w, dtype):
    """x [R,I], w [O,I] in float64 -> (y, bound)."""
    with np.errstate(invalid="ignore", over="ignore"):
        y = x @ w.T
        size = np.abs(x) @ np.abs(w).T
    return y, 1.01 * (PARTS[dtype] * x.shape[1] + 16) * 2.0 ** -24 * size + HALF_STEP[dtype] * np.abs(y) + 1e-37


def sight(n, rows, i, window, sinks):
    """The slots that new row i of a sequence of n rows sees."""
    at = n - rows + i
    return [j for j in range(at + 1) if not window or j > at - window or j < sinks]


def attention(q, key, value, lengths, scale, window, sinks, dtype):
    """q [B,R,Hq,w], key and value [B,Hkv,C,w], float64 -> (out, bound)."""
    batch, rows, heads, width = q.shape
    kv_heads, capacity = key.shape[1], key.shape[2]
    group = heads // kv_heads
    out, bound = np.zeros_like(q), np.zeros_like(q)
    u, parts = HALF_STEP[dtype], PARTS[dtype]
    for b in range(batch):
        n = min(int(lengths[b]), capacity)
        for i in range(rows):
            seen = sight(n, rows, i, window, sinks)
            if not seen:
                continue
            for h in range(heads):
                k, v = key[b, h // group, seen], value[b, h // group, seen]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = (k @ q[b, i, h]) * scale
                    off = (parts * width + 4) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(q[b, i, h]))
                    x = s - s.max()
                    e = np.exp(x)
                    p = e / e.sum()
                    rel = 2 * off.max() + 2.0 ** -23 * (np.abs(x) + 16) + 2.0 ** -21 + 2 * parts * len(seen) * 2.0 ** -23
                    if dtype == "bf16":
                        rel = rel + u
                    out[b, i, h] = p @ v
                    bound[b, i, h] = 1.01 * ((p * rel) @ np.abs(v) + u * np.abs(out[b, i, h])) + 1e-37
    return out, bound


def rotated(x, positions, theta=1e6):
    """x [..., R, H, w] at FP32 angles of positions [..., R]; the rotation in FP32, unrounded to storage."""
    width = x.shape[-1]
    exponent = (2 * np.arange(width // 2)).astype(np.float32) / np.float32(width)
    frequency = (1.0 / theta ** exponent.astype(np.float64)).astype(np.float32)
    angle = (positions.astype(np.float32)[..., None] * frequency).astype(np.float64)
    c, s = np.cos(angle).astype(np.float32)[..., None, :], np.sin(angle).astype(np.float32)[..., None, :]
    lo, hi = x[..., :width // 2].astype(np.float32), x[..., width // 2:].astype(np.float32)
    return np.concatenate((lo * c - hi * s, hi * c + lo * s), -1)
