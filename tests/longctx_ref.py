"""Plain numpy restatements, in 64 bits, of the long-context operators: rotation and norms, the 4-bit
blocks, attention with a window and visible first tokens."""
import numpy as np


def frequencies(rope_dim, base, scaling="none", factor=1.0, orig=0, low=1.0, high=4.0):
    f = float(base) ** (-2.0 * np.arange(rope_dim // 2) / max(rope_dim, 1))
    if scaling == "linear":
        return f / factor
    if scaling == "blend":
        g = np.clip((orig * f / (2 * np.pi) - low) / (high - low), 0, 1)
        return f * (g + (1 - g) / factor)
    return f


def rms(x, gamma, eps):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gamma.astype(np.float64)


def rotate(x, pos, freq, layout, magnitude=1.0):
    """x [n, heads, dim], pos [n]."""
    y = x.astype(np.float64).copy()
    p = len(freq)
    t = np.asarray(pos, np.float64)[:, None, None] * freq
    c, s = magnitude * np.cos(t), magnitude * np.sin(t)
    i, j = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if layout == "adjacent" else (slice(0, p), slice(p, 2 * p))
    a, b = y[..., i].copy(), y[..., j].copy()
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


def q40(x):
    """fp32 rows [..., D] -> blocks [..., D/32, 18] uint8, in the arithmetic of the definition (fp32)."""
    x = np.asarray(x, np.float32)
    x = x.reshape(*x.shape[:-1], -1, 32)
    hi, lo = x.max(-1), x.min(-1)
    m = np.where(hi >= -lo, hi, lo)
    d = np.clip(m * np.float32(-0.125), -65504, 65504).astype(np.float16)
    df = d.astype(np.float32)[..., None]
    inv = np.divide(np.float32(1), df, out=np.zeros_like(df), where=df != 0)
    code = np.clip(np.rint(x * inv) + 8, 0, 15).astype(np.uint8)
    return np.concatenate([d[..., None].view(np.uint8), code[..., :16] | (code[..., 16:] << 4)], -1)


def q40_values(blocks):
    """Blocks -> values [..., D] in 64 bits."""
    d = np.ascontiguousarray(blocks[..., :2]).view(np.float16).astype(np.float64)
    codes = np.concatenate([blocks[..., 2:] & 15, blocks[..., 2:] >> 4], -1).astype(np.float64) - 8
    return (codes * d).reshape(*blocks.shape[:-2], blocks.shape[-2] * 32)


def seen(p, n_keys, window, sinks):
    """Keys j < n_keys that a query at position p sees."""
    j = np.arange(n_keys)
    ok = j <= p
    if window:
        ok &= (j > p - window) | (j < sinks)
    return np.nonzero(ok)[0]


def attend(q, k, v, scale):
    """q [dim], k, v [keys, dim]: zeros without keys."""
    if len(k) == 0:
        return np.zeros(q.shape, np.float64)
    s = k.astype(np.float64) @ q.astype(np.float64) * scale
    w = np.exp(s - s.max())
    return (w / w.sum()) @ v.astype(np.float64)


def window_attention(q, k, v, pos0, lens, window, sinks, scale):
    """q [B, n, H, D], k, v [B, m, Hk, D]."""
    B, n, H, D = q.shape
    group = H // k.shape[2]
    out = np.zeros(q.shape, np.float64)
    for b in range(B):
        for i in range(n):
            keys = seen(int(pos0[b]) + i, min(int(lens[b]), k.shape[1]), window, sinks)
            for h in range(H):
                out[b, i, h] = attend(q[b, i, h], k[b, keys, h // group], v[b, keys, h // group], scale)
    return out
