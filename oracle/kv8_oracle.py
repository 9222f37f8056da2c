"""The 8-bit K/V cache on the CPU: the written codes and scales by the definition's fp32 arithmetic, and the
cache's values and attention over it in float64."""

import numpy as np

BLOCK = 64
TOP = {"int8": 127.0, "e4m3": 448.0}


def round_e4m3(x):
    """float values -> the nearest e4m3 values (3 mantissa bits, least exponent -6, ties to even), saturated."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    with np.errstate(divide="ignore"):
        e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
    step = 2.0 ** (e - 3)
    return np.sign(x) * np.minimum(np.rint(a / step) * step, 448.0)


def _round(x, fmt):
    x = np.clip(x, -TOP[fmt], TOP[fmt])
    return np.rint(x).astype(np.float64) if fmt == "int8" else round_e4m3(x)


def write(values, scale, x, fmt, start, count):
    """One sequence and head: ``values`` [capacity, dim] (code values, float64), ``scale`` [blocks] float32 and new
    rows ``x`` [tokens, dim] fp16.  Returns the updated copies."""
    values, scale = values.copy(), scale.copy()
    cap = values.shape[0]
    one = np.float32(1)
    first, end = max(start, 0), min(start + min(max(count, 0), x.shape[0]), cap)
    for blk in range(first // BLOCK, -(-end // BLOCK)):
        lo, hi = max(first, blk * BLOCK), min(end, (blk + 1) * BLOCK)
        if lo >= hi:
            continue
        new = x[lo - start:hi - start].astype(np.float32)
        a = np.abs(new[np.isfinite(new)]).max(initial=np.float32(0))
        s = np.float32(a) * (one / np.float32(TOP[fmt]))
        held = lo > blk * BLOCK
        before = scale[blk]
        if held:
            s = max(s, before)
        inv = one / s if s > 0 else np.float32(0)
        with np.errstate(invalid="ignore", over="ignore"):
            scaled = np.where(np.isnan(new), np.float32(0), new) * inv
        codes = np.zeros(new.shape) if s == 0 else _round(scaled, fmt)
        if held and s > before:
            f = before * inv
            values[blk * BLOCK:lo] = _round(values[blk * BLOCK:lo].astype(np.float32) * f, fmt)
        values[lo:hi] = codes
        scale[blk] = s
    return values, scale


def decode(values, scale):
    """[..., capacity, dim] code values and [..., blocks] scales -> float64."""
    n = values.shape[-2]
    s = np.repeat(np.asarray(scale, np.float64), BLOCK, axis=-1)[..., :n]
    return values * s[..., None]


def attention(q, k, v, lens, causal=False, scale=None):
    """q [B, S, H, D], k and v [B, Hkv, L, D] float64, lens[b] tokens of each sequence -> [B, S, H, D] float64."""
    q = np.asarray(q, np.float64)
    b, n_q, h, d = q.shape
    group = h // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = np.zeros(q.shape)
    for i in range(b):
        n = int(lens[i])
        if n == 0:
            continue
        for a in range(h):
            s = q[i, :, a] @ k[i, a // group, :n].T * scale
            if causal:
                pos = n - n_q + np.arange(n_q)
                s = np.where(np.arange(n)[None, :] <= pos[:, None], s, -np.inf)
            top = s.max(1, keepdims=True)
            live = np.isfinite(top[:, 0])
            p = np.exp(s[live] - top[live])
            out[i, live, a] = p @ v[i, a // group, :n] / p.sum(1, keepdims=True)
    return out
