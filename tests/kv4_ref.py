"""Plain restatements in 64 bits of the operators around the 4-bit cache (numpy, CPU)."""
import numpy as np


def quantise(x):
    """Values [..., d] (any float type) -> the cache's values for them, as float64: a scale per 32, eight significant bits."""
    h = np.asarray(x).astype(np.float16)
    g = h.astype(np.float64).reshape(*h.shape[:-1], -1, 32)
    top = np.abs(g).max(-1, keepdims=True)
    step = round_to_8_bits((top.astype(np.float32) / np.float32(7)).astype(np.float32)).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        code = np.where(step > 0, np.clip(np.rint(g / step), -7, 7), 0.0)
    out = code * step
    out[~np.isfinite(g).all(-1)] = np.nan
    return out.reshape(h.shape)


def round_to_8_bits(x):
    """float32 -> the nearest float32 with eight significant bits, ties to even."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    return u.astype(np.uint32).view(np.float32)


def norm_rope(x, weight, eps, positions, rotary, neighbours, sections, min_ts, max_ts):
    """x [tokens][heads][d], positions [axes][tokens] -> float64."""
    x = np.asarray(x, np.float64).copy()
    if weight is not None:
        x *= np.asarray(weight, np.float64) / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    half = rotary // 2
    axis = np.repeat(np.arange(len(sections)), sections)
    for i in range(half):
        angle = np.asarray(positions)[axis[i]].astype(np.float64) / (min_ts * (max_ts / min_ts) ** (2.0 * i / rotary))
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        u, v = x[..., a].copy(), x[..., b].copy()
        x[..., a], x[..., b] = u * c - v * s, v * c + u * s
    return x


def attention(q, keys, values, queries, scale, window):
    """One sequence: q [queries][heads][d], keys / values [n][kv_heads][d] -> (o, sum of p |v|), float64, zeros where nothing is seen."""
    q, keys, values = (np.asarray(a, np.float64) for a in (q, keys, values))
    n, hk, d = keys.shape
    g = q.shape[1] // hk
    o, size = np.zeros_like(q), np.zeros_like(q)
    for i in range(queries):
        at = n - queries + i
        lo = max(0, at - window + 1) if window else 0
        if at < lo:
            continue
        for h in range(q.shape[1]):
            k, v = keys[lo:at + 1, h // g], values[lo:at + 1, h // g]
            s = k @ q[i, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h], size[i, h] = p @ v, p @ np.abs(v)
    return o, size
