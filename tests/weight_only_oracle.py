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


def product(a, w):
    """(y, bound) of a . w^T: n f32 additions of exact or once rounded products, each partial sum
    at most sum |a w|, err by (n + 2) 2^-24 sum |a w|; scaling a sum rounds once more."""
    a = a.astype(np.float64)
    return a @ w.T, (a.shape[1] + 8) * U * (np.abs(a) @ np.abs(w).T)


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
