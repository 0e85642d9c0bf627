"""How many bits of an activation the weight-only products keep beside larger ones of its row.

Rows whose blocks of 128 hold a few activations far below the rest (2^-20 to 2^-45 of it), and channels whose
only nonzero codes meet those few: nothing else reaches such an output, so what the path dropped of them shows. Each
shape reaches another kernel."""
import numpy as np
import pytest

from aikit_amd import enchip
from weight_only_bound import product
from weight_only_oracle import U, values4

pytestmark = pytest.mark.gpu

K, GROUP = 384, 64
BG = np.float32(32.0)  # silu(32) = 32 (1 - 1.3e-14)
# rows, channels: few rows in f32, pieces of 8 and of 4 wavefronts, tiles of 32 and 64 rows with K in two, and of 64
SHAPES = [(3, 300), (20, 300), (300, 1000), (600, 1000), (1100, 1200), (2100, 2000)]


def rows(g, M, small):
    """Activations of about 1e10, except `small` of each 128, which are `down` times that."""
    a = g.standard_normal((M, K))
    a = np.where(np.abs(a) < 0.1, 0.5, a) * 1e10
    at = np.concatenate([b + g.choice(128, size=small, replace=False) for b in range(0, K, 128)])
    a[:, at] *= 2.0 ** -g.integers(20, 46, size=(M, 1))
    return a.astype(np.float32), at


def codes(g, N, at, lo):
    """Channel n: one small activation (n % 4 == 0), all of them (1), one anywhere (2), all codes (3)."""
    q = np.zeros((N, K), np.int64)
    for n in range(N):
        if n % 4 == 0:
            q[n, g.choice(at)] = g.choice([1, -1, 3, lo])
        elif n % 4 == 1:
            q[n, at] = g.integers(lo, -lo, size=len(at))
        elif n % 4 == 2:
            q[n, g.integers(0, K)] = g.choice([1, -1, 3, lo])
        else:
            q[n] = g.integers(lo, -lo, size=K)
    return q


@pytest.mark.parametrize("small", [1, 8])
@pytest.mark.parametrize("M,N", SHAPES)
def test_small_activations_beside_large_ones_q4(ctx, M, N, small):
    g = np.random.default_rng(M + small)
    a, at = rows(g, M, small)
    c = (codes(g, N, at, -8) + 8).astype(np.uint8)
    s = g.uniform(0.002, 0.01, size=(N, K // GROUP)).astype(np.float16)
    h = ctx.register_weight4(c[:, 0::2] | (c[:, 1::2] << 4), s, K, GROUP)
    try:
        print(f"[case] matmul_bt_q4 M={M} N={N} small={small}", flush=True)
        got = ctx.matmul_bt_q4(h, a)
    finally:
        ctx.release_weight4(h)
    want, tol = product(a, values4(c, s, GROUP))
    assert np.all(np.abs(got - want) <= tol), f"{np.max(np.abs(got - want) / tol)} of the bound"
    lone = np.abs(got[:, ::4] - want[:, ::4])  # one activation each: the gate of f32 products
    assert np.all(lone <= 2e-4 * np.maximum(np.abs(want[:, ::4]), 1))


@pytest.mark.parametrize("form", ["q8", "q4"])
@pytest.mark.parametrize("M,N", SHAPES)
def test_small_activations_beside_large_ones_gated(ctx, form, M, N):
    # the gate's codes are 0 and its biases 32: the output is 32 times the up projection
    g = np.random.default_rng(M)
    a, at = rows(g, M, 8)
    q = codes(g, N, at, -8 if form == "q4" else -127)
    none = np.full(N, BG, np.float32)
    if form == "q4":
        s = g.uniform(0.002, 0.01, size=(N, K // GROUP)).astype(np.float16)
        pack = [(c[:, 0::2] | (c[:, 1::2] << 4)) for c in (np.full((N, K), 8, np.uint8), (q + 8).astype(np.uint8))]
        h = [ctx.register_weight4(c, s, K, GROUP) for c in pack]
        w = values4(q + 8, s, GROUP)
    else:
        s = g.uniform(0.0005, 0.002, size=N).astype(np.float32)
        h = [ctx.register_weight(c, s) for c in (np.zeros((N, K), np.int8), q.astype(np.int8))]
        w = q * s.astype(np.float64)[:, None]
    try:
        print(f"[case] gated {form} M={M} N={N}", flush=True)
        got = (ctx.gated_q4 if form == "q4" else ctx.gated_q8)(h[0], h[1], a, none, None, enchip.ACT_SILU)
    finally:
        for x in h:
            (ctx.release_weight4 if form == "q4" else ctx.release_weight)(x)
    y, tol = product(a, w)
    want, tol = 32 * y, 32 * tol + (8 + 1) * U * np.abs(32 * y)  # SiLU's 4 ulp, the product's half
    assert np.all(np.abs(got - want) <= tol * (1 + 2.0 ** -20)), f"{np.max(np.abs(got - want) / tol)} of the bound"


@pytest.mark.parametrize("M,N", SHAPES)
def test_any_spread(ctx, M, N):
    # exponents from 2^-60 to 2^60 side by side, one activation a channel
    g = np.random.default_rng(M)
    x = g.standard_normal((M, K))
    a = np.ldexp(np.where(np.abs(x) < 0.1, 0.5, x), g.integers(-60, 61, size=(M, K))).astype(np.float32)
    a[::7, ::3] = 0
    c = np.full((N, K), 8, np.uint8)
    c[np.arange(N), g.integers(0, K, size=N)] = 8 + g.choice([1, -1, 5, -8], size=N)
    s = g.uniform(0.002, 0.01, size=(N, K // GROUP)).astype(np.float16)
    h = ctx.register_weight4(c[:, 0::2] | (c[:, 1::2] << 4), s, K, GROUP)
    try:
        print(f"[case] matmul_bt_q4 spread M={M} N={N}", flush=True)
        got = ctx.matmul_bt_q4(h, a)
    finally:
        ctx.release_weight4(h)
    want, tol = product(a, values4(c, s, GROUP))
    assert np.all(np.abs(got - want) <= tol), f"{np.max(np.abs(got - want) / tol)} of the bound"


@pytest.mark.parametrize("M", [20, 300, 2100])
def test_rows_of_the_smallest_and_largest_floats(ctx, M):
    # rows whose largest is subnormal, the least normal, near f32's largest, or 0
    N = 200
    g = np.random.default_rng(M)
    x = g.standard_normal((M, K))
    top = np.array([2.0 ** -146, 2.0 ** -130, 2.0 ** -126, 1e-30, 1e30, 1e36, 0.0])[np.arange(M) % 7]
    a = (x * top[:, None]).astype(np.float32)
    c = np.full((N, K), 8, np.uint8)
    c[np.arange(N), g.integers(0, K, size=N)] = 8 + g.choice([1, -1, 5, -8], size=N)
    s = np.ones((N, K // GROUP), np.float16)
    h = ctx.register_weight4(c[:, 0::2] | (c[:, 1::2] << 4), s, K, GROUP)
    try:
        got = ctx.matmul_bt_q4(h, a)
    finally:
        ctx.release_weight4(h)
    want, tol = product(a, values4(c, s, GROUP))
    assert np.all(np.abs(got - want) <= tol + 2.0 ** -150)  # an output that is subnormal itself
