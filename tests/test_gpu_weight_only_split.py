"""The weight-only products whose rows go through the context's scratch in f16 parts: rows too long to be
held in registers, more rows than one pass takes, and the scratch limit."""
import numpy as np
import pytest

from aikit_amd import enchip
from test_gpu_gated import Pair, activations
from weight_only_oracle import product, weight4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [17, 70, 600])
@pytest.mark.parametrize("N,K,group", [(70, 4100, 96), (300, 4097, 32), (257, 8192, 128), (40, 20001, 1024)])
def test_long_rows_q4(ctx, M, N, K, group):
    g = np.random.default_rng(K + M)
    c, s, w = weight4(g, N, K, group)
    a = activations(g, M, K)
    a[3, 5] = 1e12  # a row whose other blocks are added in f32
    a[M - 1] = 0
    h = ctx.register_weight4(c, s, K, group)
    try:
        print(f"[case] matmul_bt_q4 M={M} N={N} K={K} group={group}", flush=True)
        got = ctx.matmul_bt_q4(h, a)
        want, tol = product(a, w)
        assert np.all(np.abs(got - want) <= tol), f"{np.nanmax(np.abs(got - want) / tol)} of the bound"
        assert np.array_equal(got, ctx.matmul_bt_q4(h, a))
    finally:
        ctx.release_weight4(h)


@pytest.mark.parametrize("form", ["q8", "q4", "w8a8"])
@pytest.mark.parametrize("M", [17, 300])
@pytest.mark.parametrize("N,K", [(70, 4100), (257, 8192)])
def test_long_rows_gated(ctx, form, M, N, K):
    g = np.random.default_rng(K + M)
    with Pair(ctx, form, g, N, K, group=64) as p:
        print(f"[case] gated {form} M={M} N={N} K={K}", flush=True)
        a = activations(g, M, K)
        a[3, 5] = 1e6
        want, tol = p.want(a, "silu")
        assert np.all(np.abs(p.run(a, "silu") - want) <= tol)


@pytest.mark.parametrize("form", ["one", "q8", "q4"])
def test_several_passes(ctx, form):
    # a pass holds 1 GiB of parts: 65536 rows of K = 4096
    import torch

    M, K, N, lda = 65536 + 70, 4096, 33, 4096 + 4
    g = np.random.default_rng(3)
    a = torch.randn((M, lda), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    d = torch.full((M + 1, N), -7.0, device="cuda")
    rows = np.concatenate([[0, 1, 31, 32, 40000], np.arange(65500, M)])
    torch.cuda.synchronize()
    print(f"[case] {form} M={M} N={N} K={K}", flush=True)
    if form == "one":
        c, s, w = weight4(g, N, K, 64)
        h = ctx.register_weight4(c, s, K, 64)
        try:
            ctx.matmul_bt_q4_dev(h, a.data_ptr(), lda, M, d.data_ptr(), N)
            torch.cuda.synchronize()
        finally:
            ctx.release_weight4(h)
        want, tol = product(a[rows, :K].cpu().numpy(), w)
    else:
        with Pair(ctx, form, g, N, K, group=64, bias=False) as p:
            p.call_dev(p.h[0], p.h[1], a.data_ptr(), lda, M, 0, 0, enchip.ACT_GELU, d.data_ptr(), N)
            torch.cuda.synchronize()
            want, tol = p.want(a[rows, :K].cpu().numpy(), "gelu")
    got = d.cpu().numpy()
    assert np.all(np.abs(got[rows] - want) <= tol)
    assert np.all(got[M] == -7.0) and not np.any(got[:M] == -7.0)


@pytest.mark.parametrize("form", ["q8", "q4", "w8a8"])
def test_scratch_limit_declines(form):
    with enchip.Context(0) as c:
        g = np.random.default_rng(4)
        with Pair(c, form, g, 64, 512) as p:
            a = activations(g, 600, 512)
            c.set_scratch_limit(100000)  # less than any of the call's buffers
            with pytest.raises(enchip.EnchipError) as e:
                p.run(a, "silu")
            assert e.value.code == enchip.ERR_OOM
            assert np.isfinite(p.run(a[:1], "silu")).all()
            c.set_scratch_limit(0)
            want, tol = p.want(a, "silu")
            assert np.all(np.abs(p.run(a, "silu") - want) <= tol)
