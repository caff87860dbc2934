"""64-bit definitions of the batch attention and cache operations, written
row by row from their formulas, and the error bounds of the tests.

Bounds.  u is half a step of the storage type (BF16 2^-8, FP32 2^-24), all
relative.  A score is a chain of `width` FP32 products and sums: off by at
most (width + 4) 2^-24 of scale * sum |q k|.  Its exponential is off by that,
by the exponent's two roundings (2^-23 of the difference to the maximum) and
by two steps of the hardware's exp2; sums of n terms add n 2^-23.  BF16
storage rounds each exponential once more (u) and the output once (u)."""
import numpy as np

HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def attention(q, prefix_key, prefix_value, key, value, lengths, scale, dtype):
    """q [B,R,Hq,w], prefix [P,Hkv,w], own [B,C,Hkv,w], float64 -> (out, bound,
    received, bound): received [B,Hkv,C] is each own slot's softmax weight
    summed over rows and heads."""
    batch, rows, heads, width = q.shape
    capacity, kv_heads = key.shape[1], key.shape[2]
    group = heads // kv_heads
    out, bound = np.zeros_like(q), np.zeros_like(q)
    received, received_bound = np.zeros((batch, kv_heads, capacity)), np.zeros((batch, kv_heads, capacity))
    u = HALF_STEP[dtype]
    for b in range(batch):
        n = min(int(lengths[b]), capacity)
        for i in range(rows):
            own = min(max(n - rows + i + 1, 0), n)
            for h in range(heads):
                kvh = h // group
                k = np.concatenate((prefix_key[:, kvh], key[b, :own, kvh]))
                v = np.concatenate((prefix_value[:, kvh], value[b, :own, kvh]))
                if not len(k):
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    s = (k @ q[b, i, h]) * scale
                    off = (width + 4) * 2.0 ** -24 * abs(scale) * (np.abs(k) @ np.abs(q[b, i, h]))
                    x = s - s.max()
                    e = np.exp(x)
                    p = e / e.sum()
                    rel = 2 * off.max() + 2.0 ** -23 * (np.abs(x) + 16) + 2.0 ** -21 + 2 * len(k) * 2.0 ** -23
                    if dtype == "bf16":
                        rel_out = rel + u
                    else:
                        rel_out = rel
                    out[b, i, h] = p @ v
                    bound[b, i, h] = 1.01 * ((p * rel_out) @ np.abs(v) + u * np.abs(out[b, i, h])) + 1e-37
                    received[b, kvh, :own] += p[len(prefix_key):]
                    received_bound[b, kvh, :own] += 1.01 * (p * rel)[len(prefix_key):] + 1e-37
    received_bound += received * (rows * group) * 2.0 ** -24
    return out, bound, received, received_bound


def evict(weights, slots, n, budget, sinks, recent):
    """(source of every slot of the cut head, by slot) for one head's rows."""
    if n <= budget:
        return list(range(n))
    newest = max(int(p) for p in slots[:n])

    def order(s):
        p, w = int(slots[s]), float(weights[s])
        safe = p < sinks or p > newest - recent
        return (not safe, 0.0 if safe else (np.inf if np.isnan(w) else -w), s)

    kept = set(sorted(range(n), key=order)[:budget])
    fill = iter(sorted(s for s in kept if s >= budget))
    return [s if s in kept else next(fill) for s in range(budget)]
