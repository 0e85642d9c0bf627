"""Every tile kernel of the weight-only products (256 CUs: the number of 32 x 32 pieces and the scale group choose
it), with rows that are added in f32 in both row blocks of a tile and a last row block that is not whole."""
import numpy as np
import pytest

from test_gpu_gated import Pair
from weight_only_bound import product
from weight_only_oracle import U, gated, values4, weight4

pytestmark = pytest.mark.gpu

# M, K, N, group: 1025 to 3840 pieces (32-row tiles, K in two), scales shared by 1 and 2 chunks; more (64-row
# tiles), scales shared by 1, 2 and 4; last groups and last blocks of 128 that are not whole
ONE = [(1000, 288, 1300, 32), (1000, 288, 1300, 96), (515, 1024, 4100, 64), (1000, 1000, 1300, 128), (1000, 1001, 1300, 64),
       (4100, 288, 1024, 32), (4100, 1000, 1024, 96), (4100, 288, 1024, 64), (4100, 1001, 1024, 64), (4100, 256, 1024, 128),
       (4100, 1000, 1024, 128), (4100, 416, 1024, 256)]
# pairs: 513 to 1024 pieces (32-row tiles, K in two), up to 2560 (64-row tiles, K in two), more (64-row tiles)
PAIRS = [(m, k, 1000, gr) for m in (600, 1500, 3000) for k, gr in ((288, 32), (1000, 96), (1001, 64), (288, 128))]


def spiked(g, M, K, tops):
    """Ordinary rows, every third of which holds one value far above the rest; and where those are."""
    a = g.standard_normal((M, K)).astype(np.float32)
    r = np.arange(0, M, 3)
    at = g.integers(0, K, size=len(r))
    a[r, at] = g.choice(np.array(tops, np.float32), size=len(r))
    a[M - 1, 0] = tops[0]
    return a, at


@pytest.mark.parametrize("M,K,N,group", ONE)
def test_products(ctx, M, K, N, group):
    g = np.random.default_rng(M + K + group)
    a, _ = spiked(g, M, K, [1e9, -1e12, 1e30])
    c, s, _ = weight4(g, N, K, group)
    q = np.stack([c & 15, c >> 4], axis=2).reshape(N, -1)
    q[::2, g.permutation(K)[:K // 2]] = 8  # half of the channels miss half of the spikes
    h = ctx.register_weight4(q[:, 0::2] | (q[:, 1::2] << 4), s, K, group)
    try:
        print(f"[case] matmul_bt_q4 M={M} K={K} N={N} group={group}", flush=True)
        got = ctx.matmul_bt_q4(h, a)
        want, tol = product(a, values4(q[:, :K], s, group))
        assert np.all(np.abs(got - want) <= tol), f"{np.max(np.abs(got - want) / tol)} of the bound"
        assert np.array_equal(got, ctx.matmul_bt_q4(h, a))
        plain = ~(np.abs(a) > 1e8).any(axis=1)  # a row's outputs do not depend on its neighbours
        assert np.array_equal(ctx.matmul_bt_q4(h, np.where(plain[:, None], a, 0))[plain], got[plain])
    finally:
        ctx.release_weight4(h)


@pytest.mark.parametrize("form,M,K,N,group", [("q4", *p) for p in PAIRS] +
                         [("q8", m, k, 1000, 0) for m in (600, 1500, 3000) for k in (288, 1001)])
def test_pairs(ctx, form, M, K, N, group):
    g = np.random.default_rng(M + K + group)
    a, _ = spiked(g, M, K, [1e9, -1e12, 1e15])
    with Pair(ctx, form, g, N, K, group=group) as p:
        print(f"[case] gated {form} M={M} K={K} N={N} group={group}", flush=True)
        y = [product(a, w) for w in p.w]
        y = [(v + b, e + U * (np.abs(v) + np.abs(b))) for (v, e), b in zip(y, p.b)]
        want, tol = gated(*y[0], *y[1], "silu")
        got = p.run(a, "silu")
        assert np.all(np.abs(got - want) <= tol), f"{np.nanmax(np.abs(got - want) / tol)} of the bound"
        assert np.array_equal(got, p.run(a, "silu"))
