"""Products with 4-bit weights and group scales (enchip_matmul_bt_q4) against float64.

Beyond the error bound of f32 sums (weight_only_oracle.product): integer activations with
power-of-two scales come out exact, and one-hot weights return single activations, so that a wrong
k order, group, channel or a dropped part of a split shows."""
import numpy as np
import pytest

from aikit_amd import enchip
from weight_only_oracle import product, values4, weight4

pytestmark = pytest.mark.gpu

MS = [1, 2, 3, 4, 5, 8, 16, 17, 33, 70]
SHAPES = [(1, 1, 32), (7, 31, 32), (16, 32, 32), (17, 33, 32), (33, 64, 64), (70, 100, 32), (257, 1000, 128), (1001, 1001, 32),
          (130, 4096, 1024), (64, 300, 512), (96, 96, 96), (300, 2050, 64)]
LARGE = [(130, 768, 1024, 64), (513, 1000, 1001, 32), (1500, 1024, 384, 128), (4100, 384, 257, 32), (300, 1536, 2304, 96)]


def say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.mark.parametrize("N,K,group", SHAPES)
def test_against_float64(ctx, N, K, group):
    g = np.random.default_rng(N * 7 + K)
    c, s, w = weight4(g, N, K, group)
    h = ctx.register_weight4(c, s, K, group)
    try:
        assert ctx.weight4_shape(h) == (N, K, group)
        for M in MS:
            say(f"matmul_bt_q4 M={M} N={N} K={K} group={group}")
            a = (g.standard_normal((M, K)) * np.where(g.random((M, K)) < 0.01, 20, 1)).astype(np.float32)
            got = ctx.matmul_bt_q4(h, a)
            want, tol = product(a, w)
            assert np.all(np.abs(got - want) <= tol), f"{np.max(np.abs(got - want) / tol)} of the bound"
            assert np.array_equal(got, ctx.matmul_bt_q4(h, a))
    finally:
        ctx.release_weight4(h)


@pytest.mark.parametrize("M,K,N,group", LARGE)
def test_many_rows(ctx, M, K, N, group):
    g = np.random.default_rng(M)
    c, s, w = weight4(g, N, K, group)
    h = ctx.register_weight4(c, s, K, group)
    try:
        say(f"matmul_bt_q4 M={M} N={N} K={K} group={group}")
        a = g.standard_normal((M, K)).astype(np.float32)
        got = ctx.matmul_bt_q4(h, a)
        want, tol = product(a, w)
        assert np.all(np.abs(got - want) <= tol)
    finally:
        ctx.release_weight4(h)


@pytest.mark.parametrize("M", [1, 2, 4, 7, 40, 200, 1100])
@pytest.mark.parametrize("N,K,group", [(70, 100, 32), (300, 1000, 64), (33, 4096, 128), (1001, 1001, 32), (64, 31, 32)])
def test_exact_on_integers(ctx, M, N, K, group):
    # |a| <= 16, |q| <= 8: every partial sum of 4096 products is an integer multiple of the
    # smallest scale below 2^24 of it (scales 1/2, 1, 2: 16 * 8 * 4096 * 4 = 2^21 halves)
    g = np.random.default_rng(M + N)
    c = g.integers(0, 16, size=(N, K + K % 2)).astype(np.uint8)
    s = np.ldexp(1.0, g.integers(-1, 2, size=(N, -(-K // group)))).astype(np.float16)
    a = g.integers(-16, 17, size=(M, K)).astype(np.float32)
    h = ctx.register_weight4(c[:, 0::2] | (c[:, 1::2] << 4), s, K, group)
    try:
        say(f"matmul_bt_q4 integers M={M} N={N} K={K} group={group}")
        assert np.array_equal(ctx.matmul_bt_q4(h, a), (a.astype(np.float64) @ values4(c[:, :K], s, group).T).astype(np.float32))
    finally:
        ctx.release_weight4(h)


@pytest.mark.parametrize("M", [1, 3, 6, 20, 50, 300, 2100])
@pytest.mark.parametrize("spread", [1, 8, 25])
def test_one_hot_selects_activations(ctx, M, spread):
    # one nonzero code per channel: the output is one activation times a power of two and a scale,
    # to the bits that the path holds of it, whatever stands beside it (over 1e-25 .. 1e25 too)
    N, K, group = 300, 300, 32
    g = np.random.default_rng(M)
    x = g.standard_normal((M, K))
    a = (np.where(np.abs(x) < 0.1, 0.5, x) * 10.0 ** g.integers(-spread, spread + 1, size=(M, K))).astype(np.float32)
    at, q = g.integers(0, K, size=N), g.choice(np.array([1, -1, 2, 4, -4, -8]), size=N)
    c = np.full((N, K), 8, np.uint8)
    c[np.arange(N), at] = q + 8
    s = np.ldexp(1.0, g.integers(-4, 4, size=(N, -(-K // group)))).astype(np.float16)
    h = ctx.register_weight4(c[:, 0::2] | (c[:, 1::2] << 4), s, K, group)
    try:
        say(f"matmul_bt_q4 one-hot M={M} spread={spread}")
        got = ctx.matmul_bt_q4(h, a)
        want, tol = product(a, values4(c, s, group))
        assert np.all(np.abs(got - want) <= tol), f"{np.max(np.abs(got - want) / tol)} of the bound"
        if M <= 6:  # rows few enough for f32 products
            assert np.array_equal(got, want.astype(np.float32))
    finally:
        ctx.release_weight4(h)


@pytest.mark.parametrize("M", [20, 300, 2100])
def test_spikes_leave_their_neighbours(ctx, M):
    # one value of 1e30 or 1e-30 among ordinary ones, and channels whose code there is 0
    N, K, group = 200, 512, 32
    g = np.random.default_rng(M)
    c, s, _ = weight4(g, N, K, group)
    codes = np.stack([c & 15, c >> 4], axis=2).reshape(N, K)
    a = g.standard_normal((M, K)).astype(np.float32)
    at = g.integers(0, K, size=M)
    a[np.arange(M), at] = g.choice(np.array([1e30, -1e30, 1e-30, 1e9, 3e4], np.float32), size=M)
    codes[::2, np.unique(at)] = 8
    h = ctx.register_weight4(codes[:, 0::2] | (codes[:, 1::2] << 4), s, K, group)
    try:
        got = ctx.matmul_bt_q4(h, a)
        want, tol = product(a, values4(codes, s, group))
        assert np.all(np.abs(got - want) <= tol), f"{np.max(np.abs(got - want) / tol)} of the bound"
    finally:
        ctx.release_weight4(h)


@pytest.mark.parametrize("M", [1, 4, 40, 300])
def test_non_finite_activations(ctx, M):
    N, K, group = 96, 200, 64
    g = np.random.default_rng(5)
    c, s, w = weight4(g, N, K, group)
    a = g.standard_normal((M, K)).astype(np.float32)
    a[0, 5], a[M // 2, 199], a[M - 1, 7] = np.inf, -np.inf, np.nan
    h = ctx.register_weight4(c, s, K, group)
    try:
        got = ctx.matmul_bt_q4(h, a)
    finally:
        ctx.release_weight4(h)
    with np.errstate(invalid="ignore"):
        want = a.astype(np.float64) @ w.T
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    fin = np.isfinite(want)
    assert np.all(np.abs(got[fin] - want[fin]) <= product(np.nan_to_num(a, nan=0, posinf=0, neginf=0), w)[1][fin])


@pytest.mark.parametrize("M", [1, 3, 5, 33, 200, 700])
@pytest.mark.parametrize("K,pad,off", [(768, 4, 0), (100, 3, 1), (33, 0, 0), (64, 1, 3), (1024, 0, 2)])
def test_dev_pitches(ctx, M, K, pad, off):
    import torch

    N, group = 200, 32
    g = np.random.default_rng(K + M)
    c, s, w = weight4(g, N, K, group)
    a = g.standard_normal((M, K)).astype(np.float32)
    h = ctx.register_weight4(c, s, K, group)
    try:
        say(f"matmul_bt_q4_dev M={M} K={K} pad={pad} off={off}")
        buf = torch.full((M * (K + pad) + off,), float("nan"), device="cuda")
        da = buf[off:].view(M, K + pad)
        da[:, :K] = torch.from_numpy(a).cuda()
        dd = torch.full((M + 2, N + 5), -7.0, device="cuda")
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        ctx.matmul_bt_q4_dev(h, da.data_ptr(), K + pad, M, dd.data_ptr(), N + 5, stream=st.cuda_stream)
        st.synchronize()
        got = dd.cpu().numpy()
        want, tol = product(a, w)
        assert np.all(np.abs(got[:M, :N] - want) <= tol)
        assert np.all(got[:, N:] == -7.0) and np.all(got[M:] == -7.0)
    finally:
        ctx.release_weight4(h)


def test_refusals(ctx):
    import torch

    g = np.random.default_rng(1)
    c, s, _ = weight4(g, 40, 100, 32)
    for kw in (dict(group=16), dict(group=48), dict(group=0), dict(group=1 << 21)):
        with pytest.raises((enchip.EnchipError, ValueError)):
            ctx.register_weight4(c, s if kw["group"] else s, 100, kw["group"])
    for bad in (np.inf, -np.inf, np.nan):
        t = s.copy()
        t[39, 3] = bad
        with pytest.raises(enchip.EnchipError, match="not finite"):
            ctx.register_weight4(c, t, 100, 32)
    with pytest.raises(ValueError):
        ctx.register_weight4(c[:, :-1], s, 100, 32)
    with pytest.raises(ValueError):
        ctx.register_weight4(c, s[:, :-1], 100, 32)
    lib, out = enchip.load(), np.zeros(1, np.uint64)
    for N, K in ((0, 32), (1, 0), (-1, 32), (1, 200000), ((1 << 24) + 1, 32), (1 << 24, 131072)):
        import ctypes

        rc = lib.enchip_weight4_register(ctx.handle, c.ctypes.data, s.ctypes.data, N, K, 32,
                                         out.ctypes.data_as(ctypes.POINTER(ctypes.c_uint64)))
        assert rc == enchip.ERR_ARG and out[0] == 0, (N, K)
    h = ctx.register_weight4(c, s, 100, 32)
    d = torch.zeros(64 * 100, device="cuda")
    p = d.data_ptr()
    for args in ((p, 99, 4, p, 40), (p, 100, 4, p, 39), (0, 100, 4, p, 40), (p, 100, 4, 0, 40), (p, 100, -1, p, 40),
                 (p, 100, 1 << 34, p, 40)):
        with pytest.raises(enchip.EnchipError) as e:
            ctx.matmul_bt_q4_dev(h, *args)
        assert e.value.code == enchip.ERR_ARG
    with pytest.raises(ValueError):
        ctx.matmul_bt_q4(h, np.zeros((2, 99), np.float32))
    assert ctx.matmul_bt_q4(h, np.zeros((0, 100), np.float32)).shape == (0, 40)
    w8 = ctx.register_weight(np.zeros((40, 100), np.int8), np.ones(40, np.float32))
    try:  # one kind's handle is not the other's
        with pytest.raises(enchip.EnchipError) as e:
            ctx.matmul_bt_q4_dev(enchip.Weight4(w8.handle, 40, 100, 32), p, 100, 1, p, 40)
        assert e.value.code == enchip.ERR_HANDLE
        with pytest.raises(enchip.EnchipError) as e:
            ctx.matmul_bt_q8_dev(enchip.Weight(h.handle, 40, 100), p, 100, 1, p, 40)
        assert e.value.code == enchip.ERR_HANDLE
    finally:
        ctx.release_weight(w8)
    ctx.release_weight4(h)
    with pytest.raises(enchip.EnchipError) as e:
        ctx.release_weight4(h)
    assert e.value.code == enchip.ERR_HANDLE
