"""Plain 64-bit forms of rotary positions and of attention over a latent cache,
for the tests: numpy, one sequence and head at a time, straight from the
definitions."""

import math

import numpy as np

ROPE, NOPE, P = 64, 128, 16


def frequencies(rotary, base, scaling="none", factor=1.0, original=0, low=1.0, high=None):
    high = (4.0 if scaling == "bands" else 32.0) if high is None else high
    out = []
    for i in range(rotary // 2):
        f = base ** (-2 * i / rotary)
        if scaling == "linear":
            f /= factor
        elif scaling == "ntk":
            f = (base * factor ** (rotary / (rotary - 2))) ** (-2 * i / rotary)
        elif scaling == "ramp":
            def pair(turns):
                return rotary * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
            a = max(math.floor(pair(high)), 0)
            b = min(math.ceil(pair(low)), rotary - 1)
            w = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            f = (1 - w) * f + w * f / factor
        elif scaling == "bands":
            turns = original * f / (2 * math.pi)
            w = min(max((turns - low) / (high - low), 0.0), 1.0)
            f = (1 - w) * f / factor + w * f
        out.append(f)
    return np.array(out)


def tables(rows, rotary, base=10000.0, first=0, **scaling):
    a = (first + np.arange(rows, dtype=np.float64))[:, None] * frequencies(rotary, base, **scaling)
    return np.cos(a), np.sin(a)


def rotate32(x, cos, sin, layout, inverse=False):
    """fp32 rows [..., dim] whose first 2 * cos.shape[-1] elements turn, each product
    and sum rounded on its own."""
    r = 2 * cos.shape[-1]
    one, two = ((slice(0, r, 2), slice(1, r, 2)) if layout == "pairs"
                else (slice(0, r // 2), slice(r // 2, r)))
    a, b = x[..., one].astype(np.float32), x[..., two].astype(np.float32)
    c, s = cos.astype(np.float32), sin.astype(np.float32)
    s = -s if inverse else s
    y = x.astype(np.float32).copy()
    y[..., one] = a * c - b * s
    y[..., two] = a * s + b * c
    return y


def softmax_sum(x, v):
    """Row by row of scores [rows, keys]: the weighted mean of v [keys, dim], 0
    without keys."""
    if x.shape[1] == 0:
        return np.zeros((x.shape[0], v.shape[1]))
    w = np.exp(x - x.max(axis=1, keepdims=True))
    return (w @ v) / w.sum(axis=1, keepdims=True)


def latent_attention(q, rows, length, count, scale, latent, out):
    """One sequence: q [H, T, latent + 64], rows [>= length, latent + 64] of its
    tokens.  Fills out [H, T, latent] (float64) for t < count."""
    q, rows = q.astype(np.float64), rows.astype(np.float64)
    for t in range(min(count, q.shape[1])):
        seen = rows[:max(length - count + t + 1, 0)]
        out[:, t] = softmax_sum(q[:, t] @ seen.T * scale, seen[:, :latent])


def expanded_attention(q, k, r, v, length, count, scale, out):
    """One sequence: q [H, T, 192], k and v [H, S, 128], r [S, 64]."""
    for h in range(q.shape[0]):
        key = np.concatenate([k[h], r], axis=-1).astype(np.float64)
        for t in range(min(count, q.shape[1])):
            n = max(length - count + t + 1, 0)
            x = (q[h, t].astype(np.float64) @ key[:n].T * scale)[None]
            out[h, t] = softmax_sum(x, v[h, :n].astype(np.float64))[0]
