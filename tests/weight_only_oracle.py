"""Weights, float64 results and error bounds for the 4-bit products and the gated projections."""
import numpy as np

U = 2.0 ** -24  # half a step of f32, relative


def weight4(g, N, K, group, lo=0):
    """Random codes [N, ceil(K/2)] and f16 scales [N, ceil(K/group)], and the values [N, K] in
    float64. An odd K's unused half byte holds a code too."""
    c = g.integers(lo, 16, size=(N, K + K % 2)).astype(np.uint8)
    s = g.uniform(0.002, 0.01, size=(N, -(-K // group))).astype(np.float16)
    return c[:, 0::2] | (c[:, 1::2] << 4), s, values4(c[:, :K], s, group)


def values4(c, s, group):
    return (c.astype(np.float64) - 8) * np.repeat(s.astype(np.float64), group, axis=1)[:, :c.shape[1]]


def weight8(g, N, K):
    q = g.integers(-128, 128, size=(N, K)).astype(np.int8)
    s = g.uniform(0.0005, 0.002, size=N).astype(np.float32)
    return q, s, q.astype(np.float64) * s.astype(np.float64)[:, None]


def held(a):
    """How far an activation may be from what the path holds of it. Each row is scaled by the power of
    two that brings its largest to 2^14 .. 2^15 and split into two f16 parts: 22 bits of an
    activation (2^-22: hi truncated, what is left rounded to 11 bits), or half of lo's smallest step,
    2^-25 scaled, 2^-39 of the largest. Blocks of 128 with more than a sixteenth of the nonzero
    activations under 2^-5 scaled are computed in f32, scaled: half a step of a subnormal, 2^-150
    scaled, 2^-164 of the largest."""
    a = np.abs(a.astype(np.float64))
    top = a.max(axis=1, keepdims=True)
    _, e = np.frexp(top)
    x = np.ldexp(a, 15 - e)
    err = np.maximum(2.0 ** -22 * a, 2.0 ** -39 * top)
    for k in range(0, a.shape[1], 128):
        b = x[:, k:k + 128]
        marked = 16 * ((b != 0) & (b < 2.0 ** -5)).sum(axis=1) > (b != 0).sum(axis=1)
        err[marked, k:k + 128] = 2.0 ** -164 * top[marked]
    return err


def product(a, w):
    """(y, bound) of a . w^T. f32 sums: n additions of exact or once rounded products, each partial
    sum at most sum |a w|, err by (n + 8) 2^-24 sum |a w|; and what is held of the activations. A
    scaled sum that is subnormal rounds to half its step, 2^-164 of the row's largest as above, once
    per scale group of at least 32 and twice more."""
    h = held(a)
    a = a.astype(np.float64)
    K = a.shape[1]
    tiny = (K / 32 + 3) * 2.0 ** -164 * np.abs(a).max(axis=1, keepdims=True)
    return a @ w.T, (K + 8) * U * (np.abs(a) @ np.abs(w).T) + h @ np.abs(w).T + tiny


def act64(name, x):
    from scipy.special import ndtr

    with np.errstate(over="ignore", invalid="ignore"):
        return x / (1.0 + np.exp(-x)) if name == "silu" else x * ndtr(x)


def act_bound(name, x):
    """The device's error of act(x) at an f32 x: SiLU within 4 ulp (8 half steps) and whatever
    is under 2^-100; GELU 0.5 x (1 + erf) with erf within 1.5e-7 (its published bound) plus 8
    half steps."""
    x = np.abs(x)
    return x * 8 * U + 2.0 ** -100 if name == "silu" else x * (0.75e-7 + 8 * U)


def gated(yg, eg, yu, eu, act):
    """(out, bound) of act(yg) * yu for pre-activations off by at most eg and eu: act' is below
    1.13 for both."""
    a = act64(act, yg)
    ea = 1.13 * eg + act_bound(act, np.abs(yg) + eg)
    return a * yu, (np.abs(a) + ea) * eu + ea * np.abs(yu) + U * np.abs(a * yu) + 1e-37
