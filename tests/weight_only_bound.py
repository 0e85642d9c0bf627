"""The error bound of the weight-only products, whatever the number of rows and whatever else a row holds.

Past a few rows a row is scaled by a power of two and held in two f16 parts: hi, 11 bits rounded to nearest, and
what is left times 2^12, again 11 bits. What is left of an activation a is at most half of hi's step, 2^-11 of a's
power of two, so its own rounding is at most 2^-23 of that: 2^-23 |a|. That holds while hi is a normal f16 (scaled
values from 2^-14 on); the others' blocks are multiplied in f32, on the scaled values: a product or partial sum
that is subnormal there rounds by 2^-150, and the scale is at least 2^14 / (2 top)."""
import numpy as np

from weight_only_oracle import U


def product(a, w):
    """(y, bound) of a . w^T: 2^-23 of each activation, n products of a channel's nonzero weights that are added
    in f32, n + 8 roundings of a partial sum that is at most sum |a w|, and the smallest steps of scaled
    values, one per product and per scale group."""
    a = a.astype(np.float64)
    K = a.shape[1]
    n = np.minimum(K, np.count_nonzero(w, axis=1))[None, :]
    aw = np.abs(a) @ np.abs(w).T
    tiny = 2.0 ** -164 * np.abs(a).max(axis=1, keepdims=True) * (np.abs(w).sum(axis=1)[None, :] + K / 32 + 3)
    return a @ w.T, (2.0 ** -23 + (n + 8) * U) * aw + tiny
