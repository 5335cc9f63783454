"""Plain 64-bit restatement of the block-quantized KV cache and its attention (numpy), for the tests."""
import numpy as np

TINY_SCALE = np.float32(2.0 ** -126)


def quantize_block(x32):
    """(int8 q, float32 d) of the values of one block and KV head (any shape, float32)."""
    a = np.max(np.abs(x32)) if x32.size else np.float32(0)
    if not np.all(np.isfinite(x32)):
        return np.zeros(x32.shape, np.int8), np.float32(np.nan)
    d = np.float32(a) / np.float32(127)
    if d < TINY_SCALE:
        return np.zeros(x32.shape, np.int8), np.float32(0)
    inv = np.float32(1) / d
    return np.rint(x32 * inv).astype(np.int8), d


def cache_values(x32, block, upto=None):
    """float64 values the cache holds for one sequence: x32 [positions][heads][dim], all of it appended."""
    out = np.empty(x32.shape, np.float64)
    for b in range(0, len(x32), block):
        for h in range(x32.shape[1]):
            q, d = quantize_block(x32[b:b + block, h])
            out[b:b + block, h] = q.astype(np.float64) * np.float64(d)
    return out


def attention(q, k, v, start, scale, window=0):
    """(out, sum_j w_j |v_j|) in float64: q [n][H][hd] at positions start.., k/v [positions][Hkv][hd]."""
    n, H, hd = q.shape
    group = H // k.shape[1]
    out = np.zeros((n, H, hd))
    mag = np.zeros((n, H, hd))
    for i in range(n):
        p = start + i
        lo = max(0, p - window + 1) if window else 0
        for h in range(H):
            s = scale * (k[lo:p + 1, h // group] @ q[i, h])
            w = np.exp(s - np.max(s))
            w /= w.sum()
            out[i, h] = w @ v[lo:p + 1, h // group]
            mag[i, h] = w @ np.abs(v[lo:p + 1, h // group])
    return out, mag
