"""numpy restatement, in 64 bits, of the operators on narrow formats: MXFP4
(blocks of 32 values under a power of two) and the key / value cache in e4m3
(a power of two for each block of tokens of a head)."""

import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _floor_log2(x):
    return np.frexp(x)[1] - 1


def quantize_mxfp4(x):
    """x (..., cols) as (codes uint8 (..., 16 * blocks), scales uint8 (..., blocks))."""
    x = np.asarray(x, np.float64)
    pad = -x.shape[-1] % 32
    x = np.concatenate([x, np.zeros(x.shape[:-1] + (pad,))], -1).reshape(x.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(bad, 0.0, x)
    top = np.abs(x).max(-1, keepdims=True)
    e = np.where(top > 0, np.maximum(_floor_log2(top) - 2, -127), -127)
    y = np.abs(x) * np.exp2(-e.astype(np.float64))
    # nearest value, ties to the even code
    code = np.zeros(y.shape, np.int64)
    for i in range(7):
        mid = (E2M1[i] + E2M1[i + 1]) / 2
        code += (y > mid) | ((y == mid) & (i % 2 == 1))
    code += 8 * (np.signbit(x) & ~bad)
    code = code.reshape(code.shape[:-1] + (16, 2))
    codes = (code[..., 0] + 16 * code[..., 1]).astype(np.uint8)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)[..., 0]
    return codes.reshape(codes.shape[:-2] + (-1,)), scales


def dequantize_mxfp4(codes, scales, size=None):
    nibbles = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1,)).astype(np.int64)
    v = np.where(nibbles < 8, 1.0, -1.0) * E2M1[nibbles % 8]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * np.repeat(s, 32, -1))[..., :size]


def mxfp4_mm(a, a_scale, b, b_scale, bias=None):
    out = dequantize_mxfp4(a, a_scale) @ dequantize_mxfp4(b, b_scale).T
    return out if bias is None else out + np.asarray(bias, np.float64)


def e4m3(x):
    """x rounded to the nearest e4m3 value (ties to even); NaN past 464 and for what is not finite."""
    x = np.asarray(x, np.float64)
    finite = np.isfinite(x)
    a = np.where(finite, np.abs(x), 0.0)
    unit = np.exp2(np.maximum(_floor_log2(np.where(a > 0, a, 1.0)), -6).astype(np.float64) - 3)
    r = np.copysign(np.rint(a / unit) * unit, x)
    return np.where(finite & (np.abs(r) <= 448), r, np.nan)


def cache_scale(top):
    """2^e with the least e >= -126 for which top <= 448 * 2^e."""
    e = np.maximum(_floor_log2(np.where(top > 0, top, 1.0)) - 8, -126)
    e = np.where(448.0 * np.exp2(e.astype(np.float64)) < top, e + 1, e)
    return np.exp2(np.where(top > 0, e, -126).astype(np.float64))


def store_kv_cache(new, cache, scale, positions, lengths, block):
    """One of key and value: new (B, H, S, D) stored into copies of cache
    (B, H, C, D; values in units of their scale) and scale (B, H, blocks), which
    are returned.  Sequence b's first lengths[b] tokens go to positions[b] on;
    those outside of the cache are dropped."""
    new, cache, scale = np.asarray(new, np.float64), np.array(cache, np.float64), np.array(scale, np.float64)
    B, H, S, D = new.shape
    C = cache.shape[2]
    for b in range(B):
        count = min(max(int(lengths[b]), 0), S)
        lo, hi = max(int(positions[b]), 0), min(int(positions[b]) + count, C)
        for j in range(lo // block, -(-hi // block) if hi > lo else lo // block):
            p0, p1 = max(lo, j * block), min(hi, (j + 1) * block)
            for h in range(H):
                x = new[b, h, p0 - int(positions[b]) : p1 - int(positions[b])]
                a = np.abs(x)
                s = cache_scale(np.where(np.isfinite(a), a, 0.0).max(initial=0.0))
                if p0 > j * block:
                    old = scale[b, h, j]
                    if old > s:
                        s = old
                    else:
                        cache[b, h, j * block : p0] = e4m3(cache[b, h, j * block : p0] * (old / s))
                scale[b, h, j] = s
                cache[b, h, p0:p1] = e4m3(x / s)
    return cache, scale


def kv_cache_attention(q, k, v, k_scale, v_scale, lengths, block, causal, scale):
    """q (B, Hq, Sq, D), k and v (B, Hkv, C, D) in units of their scales.  A NaN of v
    reaches the rows that see its token."""
    q = np.asarray(q, np.float64)
    B, Hq, Sq, D = q.shape
    group = Hq // k.shape[1]
    out = np.zeros(q.shape)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), k.shape[2])
        at = np.arange(n)
        seen = at[None] <= (np.arange(Sq)[:, None] + n - Sq if causal else n)
        for h in range(Hq):
            g = h // group
            kk = np.asarray(k[b, g, :n], np.float64) * np.asarray(k_scale[b, g], np.float64)[at // block][:, None]
            vv = np.asarray(v[b, g, :n], np.float64) * np.asarray(v_scale[b, g], np.float64)[at // block][:, None]
            s = np.where(seen, q[b, h] @ kk.T * scale, -np.inf)
            top = s.max(-1, keepdims=True, initial=-np.inf)
            p = np.exp(s - np.where(np.isneginf(top), 0.0, top))
            total = p.sum(-1, keepdims=True)
            bad = np.isnan(vv)  # reaches the rows that see it
            with np.errstate(invalid="ignore", divide="ignore"):
                mean = np.where((seen @ bad.astype(np.float64)) > 0, np.nan, p @ np.where(bad, 0.0, vv) / total)
            out[b, h] = np.where(total == 0, 0.0, mean)
    return out
