"""Float64 forms of the attention block's operators: head norms with rotation, attention with a relative
position bias, low-rank adapters, and the W8A8 linear under them."""
import math

import numpy as np


def freqs64(rot, base=1e4):
    return base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


def head_norm_rope(x, q_heads, k_heads, hd, gq, gk, eps, pos, rot, interleaved, freqs=None, mscale=1.0):
    """x [rows, (q_heads + k_heads) hd] float64; pos [rows] or None. Returns the turned rows and the normed heads [rows, heads, hd]."""
    h = x.reshape(len(x), q_heads + k_heads, hd)
    with np.errstate(all="ignore"):
        n = h / np.sqrt((h * h).mean(axis=-1, keepdims=True) + eps)
    gain = np.concatenate([np.broadcast_to(gq, (q_heads, hd)), np.broadcast_to(gk, (k_heads, hd))]).astype(np.float64)
    n = n * gain
    y = n.copy()
    if rot:
        f = freqs64(rot) if freqs is None else freqs
        a = pos.astype(np.float64)[:, None] * f
        c, s = np.cos(a)[:, None] * mscale, np.sin(a)[:, None] * mscale
        j = np.arange(rot // 2)
        i, k = (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)
        y[..., i], y[..., k] = n[..., i] * c - n[..., k] * s, n[..., k] * c + n[..., i] * s
    return y.reshape(len(x), -1), n


def bucket_borders(buckets, max_distance):
    """The smallest distance of each bucket of one direction, in whole numbers."""
    half = buckets // 2
    e, m = half // 2, half - half // 2
    first = list(range(e))
    for j in range(m):
        n = e
        while n ** m * e ** j < e ** m * max_distance ** j:
            n += 1
        first.append(n)
    return first


def bucket_of(d, buckets, max_distance):
    first = np.array(bucket_borders(buckets, max_distance))
    d = np.asarray(d)
    return np.searchsorted(first, np.abs(d), side="right") - 1 + (buckets // 2) * (d > 0)


def attention(q, k, v, spans, heads, kv, hd, scale, bias=None, out=None):
    """q [T, heads hd], k and v [T, kv hd] float64; bias(d [n, n], head) -> [n, n]; rows of no span keep out's."""
    out = np.zeros_like(q) if out is None else out.astype(np.float64).copy()
    for s, e in spans:
        n = e - s
        if n <= 0:
            continue
        d = np.arange(n)[None, :] - np.arange(n)[:, None]
        for h in range(heads):
            g = h // (heads // kv)
            c, cg = slice(h * hd, (h + 1) * hd), slice(g * hd, (g + 1) * hd)
            y = scale * (q[s:e, c] @ k[s:e, cg].T)
            if bias is not None:
                y = y + bias(d, h)
            with np.errstate(invalid="ignore"):
                m = y.max(axis=1, keepdims=True)
                p = np.exp(y - np.where(np.isneginf(m), 0, m))
                l = p.sum(axis=1, keepdims=True)
                out[s:e, c] = np.where(l == 0, 0, (p / np.where(l == 0, 1, l)) @ v[s:e, cg])
    return out


def linear64(x, wq, ws, b=None):
    """The W8A8 linear of f32 rows: codes as the format has them, in f32 operations, then float64."""
    a = x.astype(np.float32)
    m = np.abs(a).max(axis=1)
    s = (m.astype(np.float64) / 127).astype(np.float32)
    inv = np.where(s > 0, 1.0 / np.where(s > 0, s, 1).astype(np.float64), 0).astype(np.float32)
    v = (a * inv[:, None]).astype(np.float64)
    c = np.clip(np.trunc(v + np.copysign(0.5, v)), -127, 127)
    y = (c @ wq.astype(np.float64).T) * s.astype(np.float64)[:, None] * ws.astype(np.float64)
    return y if b is None else y + b.astype(np.float64)


def adapters(a, ids, A, B, scale):
    """The adapters' part of rows a [M, K], and the sum of |products| behind each output: A [slots, r, K], B [slots, N, r]."""
    M, N = len(a), B.shape[1]
    y, mass = np.zeros((M, N)), np.zeros((M, N))
    for s in range(len(A)):
        rows = np.nonzero(ids == s)[0]
        if len(rows):
            x, As, Bs = a[rows].astype(np.float64), A[s].astype(np.float64), scale[s] * B[s].astype(np.float64)
            y[rows] = x @ As.T @ Bs.T
            mass[rows] = np.abs(x) @ np.abs(As).T @ np.abs(Bs).T
    return y, mass


def gelu64(x):
    erf = np.vectorize(math.erf)
    return 0.5 * x * (1 + erf(x * math.sqrt(0.5)))
