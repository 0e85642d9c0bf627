"""Rows without an adapter keep every bit of what they are added to: zeros of either sign."""
import numpy as np
import pytest

from aikit_amd import enchip, workloads
from test_gpu_adapters import Set, activations, add

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


def bits(x):
    return (x.cpu().numpy() if hasattr(x, "cpu") else x).view(np.int32)


@pytest.mark.parametrize("act", [enchip.ACT_NONE, enchip.ACT_GELU])
@pytest.mark.parametrize("M,K,N,rank", [
    (16, 384, 1536, 8), (7, 384, 100, 20),               # one launch
    (32, 1024, 4096, 32), (20, 1001, 64, 40),            # row-major codes, two launches
    (70, 256, 96, 16), (300, 768, 768, 40), (513, 1000, 1001, 16),  # pieces
    (5000, 256, 2048, 16), (6000, 256, 2048, 40),        # persistent tiles
])
@pytest.mark.parametrize("few", [0.0, 0.4])
def test_linear(ctx, M, K, N, rank, act, few):
    import torch

    say(f"linear_adapters zeros of either sign M={M} K={K} N={N} rank={rank} act={act} rows with adapters {few}")
    g = np.random.default_rng(M + N)
    wq, ws = workloads.quantize_weights((g.standard_normal((N, K)) * 0.03).astype(np.float32))
    wq[::3] = 0
    ws[::2] *= -1  # 0 times a negative scale is -0
    a = activations(g, M, K)
    a[1::5] = 0
    ids = np.where(g.random(M) < few, g.integers(0, 3, M), np.where(g.random(M) < 0.5, -1, 3))
    ids[0] = -1
    w = ctx.register_weight(wq, ws)
    try:
        with Set(ctx, K, N, rank, 3) as s:
            da, di = torch.from_numpy(a).cuda(), torch.from_numpy(ids.astype(np.int32)).cuda()
            out, plain = torch.full((M, N), 4.0, device="cuda"), torch.full((M, N), 5.0, device="cuda")
            torch.cuda.synchronize()
            ctx.linear_adapters_dev(w, s.h, da.data_ptr(), M, di.data_ptr(), 0, act, out.data_ptr())
            ctx.linear_dev(w, da.data_ptr(), M, 0, act, plain.data_ptr())
            torch.cuda.synchronize()
            none = (ids < 0) | (ids >= 3)
            want = bits(plain)[none]
            assert (want == np.int32(-2 ** 31)).any()  # some -0 among them
            assert np.array_equal(bits(out)[none], want)
    finally:
        ctx.release_weight(w)


@pytest.mark.parametrize("M,K,N,rank", [(5, 64, 40, 8), (100, 256, 300, 40), (2000, 100, 64, 16)])
@pytest.mark.parametrize("few", [0.0, 0.4])
@pytest.mark.parametrize("inplace", [False, True])
def test_add(ctx, M, K, N, rank, few, inplace):
    say(f"adapters_add zeros of either sign M={M} K={K} N={N} rank={rank} rows with adapters {few}")
    g = np.random.default_rng(M + N)
    ids = np.where(g.random(M) < few, g.integers(0, 3, M), -1)
    ids[0] = -1
    y = np.where(g.random((M, N)) < 0.3, np.float32(-0.0), g.standard_normal((M, N)).astype(np.float32)).astype(np.float32)
    with Set(ctx, K, N, rank, 3) as s:
        got = add(ctx, s, activations(g, M, K), ids, y, inplace=inplace)
        none = ids < 0
        assert np.array_equal(bits(np.ascontiguousarray(got[none])), bits(np.ascontiguousarray(y[none])))
