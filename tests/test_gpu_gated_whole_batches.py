"""W8A8 gated projections of many rows at widths that the persistent tiles refuse: an odd number of 64-deep stages,
outputs that are no multiple of 4."""
import numpy as np
import pytest

from test_gpu_gated import Pair, activations

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N", [(9000, 320, 768), (5001, 960, 514), (9001, 256, 1001), (4097, 316, 1003), (6000, 832, 132)])
def test_many_rows(ctx, M, K, N):
    g = np.random.default_rng(M + K)
    for act in ("silu", "gelu"):
        with Pair(ctx, "w8a8", g, N, K) as p:
            print(f"[case] gated w8a8 M={M} N={N} K={K} {act}", flush=True)
            a = activations(g, M, K)
            a[M // 3] = 0
            want, tol = p.want(a, act)
            got = p.run(a, act)
            assert np.all(np.abs(got - want) <= tol)
            assert np.array_equal(got, p.run(a, act))
