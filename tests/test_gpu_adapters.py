"""Low-rank adapters (enchip_adapters_add_dev, enchip_w8a8_linear_adapters_dev) against float64.

The tolerance per element. An inner product of n terms in f32, each term within 2^-24 of exact, is off by at most
(n + 1) 2^-24 times the sum of its terms' magnitudes, so the rows' low-rank parts are off by (K + 1) 2^-24 and
the result by (K + 1 + rank + 1 + 1) 2^-24 of sum |a| |A| |B| (the last for scale B's rounding), under
(K + rank + 4) 2^-24 with what those bounds leave out of second order. The W8A8 sum is exact, its scales and the bias round
three times, and the sum of both parts once: 2^-22 of the parts. The GELU is linalg.GELUF32 of that sum: its
slope is at most 1.13, and the oracle's own GELU is taken of the float64 sum rounded to f32 (another 2^-24)."""
import numpy as np
import pytest

import oracle
from aikit_amd import enchip, workloads
from block_oracle import adapters, linear64

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


class Set:
    def __init__(self, ctx, K, N, rank, slots, seed=0, scale=None):
        g = np.random.default_rng(seed + K * 3 + N + rank)
        self.ctx, self.K, self.N, self.rank, self.slots = ctx, K, N, rank, slots
        self.A = (g.standard_normal((slots, rank, K)) / np.sqrt(K)).astype(np.float32)
        self.B = (g.standard_normal((slots, N, rank)) * 0.1).astype(np.float32)
        self.scale = np.array([2.0 / (s + 1) for s in range(slots)] if scale is None else scale, np.float32)
        self.h = ctx.adapters(K, N, rank, slots)
        for s in range(slots):
            ctx.set_adapter(self.h, s, self.A[s], self.B[s], float(self.scale[s]))

    def __enter__(self):
        return self

    def __exit__(self, *e):
        self.ctx.release_adapters(self.h)

    def of(self, a, ids):
        y, mass = adapters(a, ids, self.A, self.B, self.scale.astype(np.float64))
        return y, mass * (self.K + self.rank + 4) * 2.0 ** -24


def activations(g, M, K):
    a = g.standard_normal((M, K)).astype(np.float32)
    return np.where(g.random((M, K)) < 0.01, a * 20, a).astype(np.float32)


def add(ctx, s, a, ids, y, lda=None, ldy=None, ldd=None, off=0, inplace=False, stream=0):
    import torch

    M = len(a)
    lda, ldy = lda or s.K, ldy or s.N
    ldd = ldy if inplace else (ldd or s.N)
    da = torch.full((off + M * lda + 4,), 1e9, device="cuda")
    da[off:off + M * lda].view(M, lda)[:, :s.K] = torch.from_numpy(a).cuda()
    dy = torch.full((M * ldy + 4,), 8.0, device="cuda")
    dy[:M * ldy].view(M, ldy)[:, :s.N] = torch.from_numpy(y).cuda()
    dd = dy if inplace else torch.full((M * ldd + 4,), 8.0, device="cuda")
    di = torch.from_numpy(ids.astype(np.int32)).cuda()
    torch.cuda.synchronize()
    ctx.adapters_add_dev(s.h, da.data_ptr() + 4 * off, lda, M, di.data_ptr(), dy.data_ptr(), ldy, dd.data_ptr(), ldd, stream)
    torch.cuda.synchronize()
    got = dd.cpu().numpy()
    body = got[:M * ldd].reshape(M, ldd)
    assert (got[M * ldd:] == 8.0).all() and (body[:, s.N:] == 8.0).all()
    return body[:, :s.N]


def some_ids(g, M, slots, run):
    return np.repeat(g.integers(-1, slots, -(-M // run)), run)[:M]


@pytest.mark.parametrize("M,K,N,rank,slots,run,k", [
    (1, 32, 32, 1, 1, 1, {}),
    (1, 1, 1, 1, 1, 1, {}),
    (16, 384, 1536, 8, 5, 16, {}),
    (33, 100, 70, 7, 3, 5, {}),
    (70, 257, 129, 16, 4, 1, {}),                              # every row another adapter
    (32, 64, 64, 17, 40, 1, {}),
    (130, 96, 96, 64, 2, 50, {}),
    (20, 64, 96, 256, 2, 7, {}),
    (300, 1000, 1001, 33, 3, 77, {}),
    (50, 130, 60, 4, 3, 9, dict(lda=133, ldy=61, ldd=67)),
    (50, 128, 60, 4, 3, 9, dict(lda=132, off=1)),              # rows that are 4-byte aligned
    (50, 128, 64, 4, 3, 9, dict(inplace=True, ldy=80)),
    (600, 64, 300, 12, 6, 100, {}),
    (4200, 300, 130, 70, 3, 90, {}),                           # more rows than a workgroup a CU
    (4200, 1100, 64, 16, 3, 90, dict(lda=1101)),
])
def test_add(ctx, M, K, N, rank, slots, run, k):
    say(f"adapters_add M={M} K={K} N={N} rank={rank} slots={slots} run={run} {k}")
    g = np.random.default_rng(M + K)
    with Set(ctx, K, N, rank, slots) as s:
        a, y, ids = activations(g, M, K), g.standard_normal((M, N)).astype(np.float32), some_ids(g, M, slots, run)
        ids[:1] = slots - 1
        got = add(ctx, s, a, ids, y, **k)
        part, tol = s.of(a, ids)
        want = y.astype(np.float64) + part
        tol = tol + 2.0 ** -23 * (np.abs(part) + np.abs(y))
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3])
        none = (ids < 0) | (ids >= slots)
        assert np.array_equal(got[none], y[none])


LINEAR = [
    (1, 64, 64, 4, 2, 1), (1, 384, 1536, 8, 5, 1), (5, 1000, 1001, 7, 3, 2), (16, 384, 1536, 8, 5, 16), (32, 768, 768, 16, 8, 1),
    (32, 100, 33, 3, 3, 1), (9, 4100, 64, 8, 2, 3), (17, 64, 40000, 4, 2, 5),
    (33, 768, 2304, 16, 4, 11), (64, 384, 384, 16, 4, 16), (70, 100, 33, 5, 3, 1), (200, 768, 768, 40, 3, 32), (513, 384, 1536, 16, 6, 100),
    (1500, 1000, 1001, 7, 3, 77), (700, 768, 3000, 20, 5, 300), (2000, 128, 1028, 8, 4, 512), (4100, 64, 2052, 16, 3, 700),
    (3000, 320, 2048, 32, 8, 1), (260, 2112, 516, 16, 3, 64), (6000, 72, 1001, 9, 3, 500),
    # every width that adapter_down holds, in few and many rows, one and several rank tiles
    (40, 256, 96, 70, 2, 9), (40, 512, 96, 20, 2, 9), (40, 1024, 64, 100, 2, 9), (40, 2048, 64, 20, 2, 9), (40, 4096, 64, 130, 2, 9),
    (4113, 250, 64, 40, 2, 200), (4113, 500, 96, 16, 3, 200), (4113, 1000, 70, 40, 3, 200), (4113, 2000, 64, 16, 3, 99),
    (4113, 2001, 64, 40, 2, 99), (4113, 4000, 64, 16, 2, 99), (4113, 4095, 64, 33, 2, 99), (4113, 5000, 64, 20, 2, 99),
]


@pytest.mark.parametrize("act", [enchip.ACT_NONE, enchip.ACT_GELU])
@pytest.mark.parametrize("M,K,N,rank,slots,run", LINEAR)
def test_linear(ctx, M, K, N, rank, slots, run, act):
    import torch

    bias = (M + N) % 2 == 0 or act == enchip.ACT_GELU
    say(f"linear_adapters M={M} K={K} N={N} rank={rank} slots={slots} run={run} act={act} bias={bias}")
    g = np.random.default_rng(M * 5 + K)
    wq, ws = workloads.quantize_weights((g.standard_normal((N, K)) * 0.03).astype(np.float32))
    b = (g.standard_normal(N) * 0.1).astype(np.float32) if bias else None
    a, ids = activations(g, M, K), some_ids(g, M, slots, run)
    ids[:1] = 0
    ids[-1:] = slots  # past the last slot: none
    a[M // 2] = 0
    w = ctx.register_weight(wq, ws)
    try:
        with Set(ctx, K, N, rank, slots) as s:
            da, di = torch.from_numpy(a).cuda(), torch.from_numpy(ids.astype(np.int32)).cuda()
            db = None if b is None else torch.from_numpy(b).cuda()
            out, plain = torch.full((M + 1, N), 4.0, device="cuda"), torch.empty((M, N), device="cuda")
            torch.cuda.synchronize()
            ctx.linear_adapters_dev(w, s.h, da.data_ptr(), M, di.data_ptr(), 0 if db is None else db.data_ptr(), act, out.data_ptr())
            ctx.linear_dev(w, da.data_ptr(), M, 0 if db is None else db.data_ptr(), act, plain.data_ptr())
            torch.cuda.synchronize()
            got, base = out.cpu().numpy(), plain.cpu().numpy()
            assert (got[M] == 4.0).all()
            got = got[:M]
            part, tol = s.of(a, ids)
    finally:
        ctx.release_weight(w)
    y = linear64(a, wq, ws, b)
    tol = tol + 2.0 ** -22 * (np.abs(part) + np.abs(y) + (0 if b is None else np.abs(b)))
    want = y + part
    if act == enchip.ACT_GELU:
        tol = 1.13 * (tol + 2.0 ** -24 * np.abs(want)) + 2.0 ** -22 * np.abs(want) + 2.0 ** -22
        want = oracle.gelu(want.astype(np.float32)).astype(np.float64).reshape(want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3])
    none = (ids < 0) | (ids >= slots)
    assert np.array_equal(got[none], base[none])


def test_small_ranks_in_a_larger_set(ctx):
    say("adapters of smaller rank, an empty slot, a slot set again")
    g = np.random.default_rng(2)
    K, N, M = 200, 90, 40
    h = ctx.adapters(K, N, 24, 4)
    try:
        a, y = activations(g, M, K), g.standard_normal((M, N)).astype(np.float32)
        A = [(g.standard_normal((r, K)) / 14).astype(np.float32) for r in (3, 24, 16)]
        B = [g.standard_normal((N, r)).astype(np.float32) for r in (3, 24, 16)]
        for s in range(3):
            ctx.set_adapter(h, s, A[s], B[s], 0.5)
        ids = np.arange(M) % 4

        class S:
            pass

        s = S()
        s.h, s.K, s.N = h, K, N
        for again in range(2):
            got = add(ctx, s, a, ids, y)
            assert np.array_equal(got[ids == 3], y[ids == 3])
            for i in range(3):
                rows = ids == i
                x = a[rows].astype(np.float64)
                want = y[rows] + 0.5 * (x @ A[i].astype(np.float64).T @ B[i].astype(np.float64).T)
                mass = 0.5 * (np.abs(x) @ np.abs(A[i]).T.astype(np.float64) @ np.abs(B[i]).T.astype(np.float64))
                tol = mass * (K + 28) * 2.0 ** -24 + 2.0 ** -22 * (np.abs(want) + np.abs(y[rows]))
                assert (np.abs(got[rows] - want) <= tol).all(), i
            A[1], B[1] = A[1][:5].copy(), B[1][:, :5].copy()
            ctx.set_adapter(h, 1, A[1], B[1], 0.5)
    finally:
        ctx.release_adapters(h)


def test_values_of_every_size(ctx):
    # an outlier beside small activations that the adapter does not read, sizes across the exponents
    say("adapters of activations across the exponents")
    g = np.random.default_rng(3)
    K, N, M, r = 96, 40, 34, 8
    with Set(ctx, K, N, r, 2) as s:
        s.A[:, :, 0] = 0
        for i in range(2):
            ctx.set_adapter(s.h, i, s.A[i], s.B[i], float(s.scale[i]))
        a = g.standard_normal((M, K)).astype(np.float32) * np.float32(2.0) ** g.integers(-60, 60, (M, 1)).astype(np.float32)
        a[:, 0] = np.float32(1e37)
        ids = np.arange(M) % 2
        y = np.zeros((M, N), np.float32)
        got = add(ctx, s, a, ids, y)
        part, tol = s.of(a, ids)
        assert (np.abs(got - part) <= tol + 2.0 ** -23 * np.abs(part)).all()


def test_not_finite_stays_in_its_row(ctx):
    say("adapters of infinite and NaN activations")
    g = np.random.default_rng(4)
    K, N, M = 64, 70, 40
    with Set(ctx, K, N, 8, 3) as s:
        a, y = activations(g, M, K), g.standard_normal((M, N)).astype(np.float32)
        ids = np.arange(M) % 3
        ids[9] = -1
        clean = add(ctx, s, a, ids, y)
        a[4, 7], a[20, 1], a[9, 3] = np.inf, np.nan, np.nan
        got = add(ctx, s, a, ids, y)
        bad = np.zeros(M, bool)
        bad[[4, 20]] = True
        assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean[~bad])


def test_rows_do_not_depend_on_their_neighbours(ctx):
    say("adapters: a row's bits alone and in a batch of other adapters")
    g = np.random.default_rng(5)
    K, N, M = 130, 200, 96
    with Set(ctx, K, N, 20, 5) as s:
        a, y, ids = activations(g, M, K), g.standard_normal((M, N)).astype(np.float32), g.integers(0, 5, M)
        got = add(ctx, s, a, ids, y)
        for r in (0, 17, 50, 95):
            assert np.array_equal(add(ctx, s, a[r:r + 1], ids[r:r + 1], y[r:r + 1])[0], got[r])


@pytest.mark.parametrize("M,K,N", [(20, 256, 512), (300, 256, 512)])
def test_graph_streams_and_scratch(ctx, M, K, N):
    import torch

    g = np.random.default_rng(6)
    wq, ws = workloads.quantize_weights((g.standard_normal((N, K)) * 0.03).astype(np.float32))
    w = ctx.register_weight(wq, ws)
    s = torch.cuda.Stream()
    try:
        with Set(ctx, K, N, 16, 4) as st:
            a, ids = torch.empty((M, K), device="cuda"), torch.zeros(M, dtype=torch.int32, device="cuda")
            y, e, z = (torch.zeros((M, N), device="cuda") for _ in range(3))
            torch.cuda.synchronize()

            def call(out, stream=s.cuda_stream):
                ctx.linear_adapters_dev(w, st.h, a.data_ptr(), M, ids.data_ptr(), 0, enchip.ACT_GELU, out.data_ptr(), stream)

            with torch.cuda.stream(s):
                a.normal_()
            call(e)
            torch.cuda.synchronize()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                call(y)
            say(f"linear_adapters M={M} captured, 3 replays with other adapters")
            for i in range(3):
                with torch.cuda.stream(s):
                    a.normal_()
                    ids.random_(-1, 4)
                torch.cuda.synchronize()
                gr.replay()
                torch.cuda.synchronize()
                call(e)
                torch.cuda.synchronize()
                assert torch.equal(y, e)
            del gr
            # two streams in turn on the shared scratch
            t = torch.cuda.Stream()
            torch.cuda.synchronize()
            for i in range(8):
                call(y, s.cuda_stream), call(z, t.cuda_stream), call(e, 0)
            torch.cuda.synchronize()
            assert torch.equal(y, z) and torch.equal(y, e)
    finally:
        ctx.release_weight(w)


def test_scratch_limit(ctx):
    import torch

    say("adapters: scratch limit")
    with Set(ctx, 64, 64, 16, 2) as s:
        a, y = torch.zeros((4096, 64), device="cuda"), torch.zeros((4096, 64), device="cuda")
        ids = torch.zeros(4096, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        ctx.set_scratch_limit(1000)
        try:
            with pytest.raises(enchip.EnchipError) as err:
                ctx.adapters_add_dev(s.h, a.data_ptr(), 64, 4096, ids.data_ptr(), y.data_ptr(), 64, y.data_ptr(), 64)
            assert err.value.code == enchip.ERR_OOM
        finally:
            ctx.set_scratch_limit(0)
        ctx.adapters_add_dev(s.h, a.data_ptr(), 64, 4096, ids.data_ptr(), y.data_ptr(), 64, y.data_ptr(), 64)
        torch.cuda.synchronize()


def test_refusals(ctx):
    import torch

    x = torch.zeros(8192, device="cuda")
    ids = torch.zeros(16, dtype=torch.int32, device="cuda")
    p, q, i = x.data_ptr(), x.data_ptr() + 16384, ids.data_ptr()
    for k in ((0, 8, 1, 1), (8, 0, 1, 1), (8, 8, 0, 1), (8, 8, 257, 1), (8, 8, 1, 0), (8, 8, 1, 65537), (131073, 8, 1, 1), (8, 2 ** 24 + 1, 1, 1),
              (131072, 2 ** 24, 256, 65536)):
        with pytest.raises(enchip.EnchipError) as err:
            ctx.adapters(*k)
        assert err.value.code == enchip.ERR_ARG, k
    wq, ws = workloads.quantize_weights(np.eye(32, 64, dtype=np.float32))
    w = ctx.register_weight(wq, ws)
    try:
        with Set(ctx, 64, 32, 4, 2) as s:
            A, B = s.A[0], s.B[0]
            for slot, a_, b_, sc in ((2, A, B, 1.0), (-1, A, B, 1.0), (0, A * np.inf, B, 1.0), (0, A, B * np.nan, 1.0), (0, A, B, np.inf),
                                     (0, A, B * 10, 3e38), (0, np.full_like(A, 2.0 ** 127), B, 1.0)):
                with pytest.raises(enchip.EnchipError) as err, np.errstate(all="ignore"):
                    ctx.set_adapter(s.h, slot, a_, B if b_ is B else b_, sc)
                assert err.value.code == enchip.ERR_ARG, slot

            assert 3e38 * np.abs(B).max() < 2.0 ** 127  # held: only scale B counts
            ctx.set_adapter(s.h, 0, A, B, 3e38)
            ctx.set_adapter(s.h, 0, A, B, 1.0)

            def add_(h=s.h, a=p, lda=64, M=4, ids=i, y=q, ldy=32, d=q, ldd=32):
                ctx.adapters_add_dev(h, a, lda, M, ids, y, ldy, d, ldd)

            def lin(w_=w, h=s.h, a=p, M=4, ids=i, act=enchip.ACT_NONE, d=q):
                ctx.linear_adapters_dev(w_, h, a, M, ids, 0, act, d)

            add_(), lin(), add_(M=0, a=0, ids=0, y=0, d=0), lin(M=0, a=0, ids=0, d=0)
            gone = enchip.Adapters(10 ** 9, 64, 32, 4, 2)
            for call, k, code in ([(add_, k, enchip.ERR_ARG) for k in (dict(a=0), dict(ids=0), dict(y=0), dict(d=0), dict(lda=63), dict(ldy=31),
                                                                       dict(ldd=31), dict(M=-1), dict(M=2 ** 30 + 1), dict(ldd=64))] +
                                  [(lin, k, enchip.ERR_ARG) for k in (dict(a=0), dict(ids=0), dict(d=0), dict(M=-1), dict(M=2 ** 30 + 1),
                                                                      dict(act=enchip.ACT_TANH), dict(act=enchip.ACT_SILU), dict(act=9))] +
                                  [(add_, dict(h=gone), enchip.ERR_HANDLE), (lin, dict(h=gone), enchip.ERR_HANDLE),
                                   (lin, dict(w_=enchip.Weight(10 ** 9, 32, 64)), enchip.ERR_HANDLE)]):
                with pytest.raises(enchip.EnchipError) as err:
                    call(**k)
                assert err.value.code == code, k
            with Set(ctx, 64, 33, 4, 1) as other, pytest.raises(enchip.EnchipError):
                lin(h=other.h)
            torch.cuda.synchronize()
    finally:
        ctx.release_weight(w)


# One launch (a's rows 16-byte aligned, K a multiple of 4 up to 1024, ranks to 32, few workgroups) and, beside it, what
# each of its limits leaves to two.
@pytest.mark.parametrize("M,K,N,rank,off", [
    (1, 4, 5, 1, 0), (7, 256, 40, 16, 0), (8, 260, 33, 17, 0), (9, 512, 64, 32, 0), (31, 516, 96, 9, 0), (32, 768, 70, 32, 0),
    (25, 772, 32, 5, 0), (32, 1024, 1024, 32, 0), (3, 1024, 4100, 8, 0),
    (16, 384, 96, 8, 1), (16, 386, 96, 8, 0), (16, 1028, 96, 8, 0), (16, 384, 96, 33, 0), (32, 128, 2304, 32, 0), (32, 64, 5000, 8, 0),
])
@pytest.mark.parametrize("act", [enchip.ACT_NONE, enchip.ACT_GELU])
def test_few_rows(ctx, M, K, N, rank, off, act):
    import torch

    say(f"linear_adapters few rows M={M} K={K} N={N} rank={rank} off={off} act={act}")
    g = np.random.default_rng(M * 7 + K + rank)
    wq, ws = workloads.quantize_weights((g.standard_normal((N, K)) * 0.03).astype(np.float32))
    b = (g.standard_normal(N) * 0.1).astype(np.float32)
    a, slots = activations(g, M, K), 5
    a[M // 3] *= np.float32(2.0 ** -40)
    ids = g.integers(-1, slots + 1, M)
    ids[M // 2] = slots - 1
    w = ctx.register_weight(wq, ws)
    try:
        with Set(ctx, K, N, rank, slots) as s:
            da = torch.empty(M * K + off, device="cuda")
            da[off:] = torch.from_numpy(a).cuda().flatten()
            di, db = torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(b).cuda()
            out, plain = torch.full((M + 1, N), 4.0, device="cuda"), torch.empty((M, N), device="cuda")

            def call(m, a_, i_, o_):
                torch.cuda.synchronize()
                ctx.linear_adapters_dev(w, s.h, a_, m, i_, db.data_ptr(), act, o_)
                torch.cuda.synchronize()

            at = da.data_ptr() + 4 * off
            call(M, at, di.data_ptr(), out.data_ptr())
            ctx.linear_dev(w, at, M, db.data_ptr(), act, plain.data_ptr())
            torch.cuda.synchronize()
            got, base = out.cpu().numpy(), plain.cpu().numpy()
            assert (got[M] == 4.0).all()
            part, tol = s.of(a, ids)
            y = linear64(a, wq, ws, b)
            tol = tol + 2.0 ** -22 * (np.abs(part) + np.abs(y) + np.abs(b))
            want = y + part
            if act == enchip.ACT_GELU:
                tol = 1.13 * (tol + 2.0 ** -24 * np.abs(want)) + 2.0 ** -22 * np.abs(want) + 2.0 ** -22
                want = oracle.gelu(want.astype(np.float32)).astype(np.float64).reshape(want.shape)
            bad = ~(np.abs(got[:M] - want) <= tol)
            assert not bad.any(), (np.argwhere(bad)[:3], got[:M][bad][:3], want[bad][:3], tol[bad][:3])
            none = (ids < 0) | (ids >= slots)
            assert np.array_equal(got[:M][none], base[none])
            # an infinite and a NaN activation leave the other rows as they were
            if M >= 7:
                torch.cuda.synchronize()
                ids[1] = ids[5] = 0
                da[off + K + K // 2], da[off + 5 * K] = float("inf"), float("nan")
                di.copy_(torch.from_numpy(ids.astype(np.int32)))
                call(M, at, di.data_ptr(), out.data_ptr())
                again = out.cpu().numpy()[:M]
                rest = [r for r in range(M) if r not in (1, 5)]
                assert np.isnan(again[[1, 5]]).all() and np.array_equal(again[rest], got[rest])
    finally:
        ctx.release_weight(w)
