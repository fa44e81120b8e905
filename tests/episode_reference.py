"""The episode memory's operators from their definitions, in 64 bits on the CPU, one world at a time."""
import math

import numpy as np

BLOCK, LARGEST, LEAST = 32, 448.0, -117


def e4m3(x):
    """x rounded to the nearest e4m3 value (ties to even); |x| <= 448."""
    a = np.abs(np.asarray(x, np.float64))
    exponent = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
    step = 2.0 ** (np.maximum(exponent, -6) - 3)
    return np.copysign(np.rint(a / step) * step, x)


def quantised(x):
    """(values, scale bytes) that x (..., head_dim) becomes in 8-bit pages."""
    x = np.asarray(x, np.float64)
    blocks = x.reshape(x.shape[:-1] + (x.shape[-1] // BLOCK, BLOCK))
    finite = np.isfinite(blocks).all(-1)
    blocks = np.where(finite[..., None], blocks, 0.0)
    most = np.abs(blocks).max(-1)
    e = np.full(most.shape, float(LEAST))
    while np.any(most > LARGEST * 2.0 ** e):
        e += most > LARGEST * 2.0 ** e
    out = e4m3(blocks * 2.0 ** -e[..., None]) * 2.0 ** e[..., None]
    out[~finite] = np.nan
    scale = np.where(finite, e + 127, 255).astype(np.uint8)
    return out.reshape(x.shape), scale


def attention(q, k, v, position, causal, window, scale):
    """One world: q (n, heads, d) at positions position .. position + n - 1, k and v (length, kv_heads, d).
    Returns out (n, heads, d), lse (n, heads), and sum p |v| (what errors of the weights scale with)."""
    n, heads, d = q.shape
    length, kv, _ = k.shape
    out, lse, size = np.zeros((n, heads, d)), np.full((n, heads), -np.inf), np.zeros((n, heads, d))
    for i in range(n):
        p = position + i
        if p < 0:
            continue
        low = max(0, p - window + 1) if window else 0
        high = min(p + 1, length) if causal else length
        if low >= high:
            continue
        for h in range(heads):
            g = h // (heads // kv)
            with np.errstate(all='ignore'):
                s = scale * (k[low:high, g] @ q[i, h])
                top = s.max() if not np.isnan(s).any() else np.nan
                if top == -np.inf:
                    continue
                w = np.exp(s - top)
                total = w.sum()
                out[i, h] = (w @ v[low:high, g]) / total
                size[i, h] = (w @ np.abs(v[low:high, g])) / total
                lse[i, h] = top + math.log(total)
    return out, lse, size
