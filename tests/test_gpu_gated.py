"""Gated projections act(a Wg^T + bg) * (a Wu^T + bu) against float64.

gated_q8 and gated_q4 within weight_only_oracle's bound of f32 sums; w8a8_gated on the linears'
own outputs, which its pre-activations equal bit for bit, so that only the gate is left."""
import numpy as np
import pytest

from aikit_amd import enchip, workloads
from weight_only_oracle import U, act64, act_bound, gated, product, weight4, weight8

pytestmark = pytest.mark.gpu

ACTS = {"silu": enchip.ACT_SILU, "gelu": enchip.ACT_GELU}
MS = [1, 2, 3, 5, 8, 16, 33, 70]
SHAPES = [(1, 1), (7, 31), (17, 33), (33, 64), (70, 100), (257, 1000), (1001, 1001), (130, 4096), (300, 768)]
LARGE = [(130, 768, 1024), (513, 1000, 1001), (1500, 1024, 384), (4100, 384, 257), (300, 1536, 2304), (2500, 128, 1536)]


def say(msg):
    print(f"[case] {msg}", flush=True)


class Pair:
    """Two registered weights of one form, their values in float64 and biases."""

    def __init__(self, ctx, form, g, N, K, group=32, bias=True):
        self.ctx, self.form, self.N, self.K = ctx, form, N, K
        made = [weight4(g, N, K, group) if form == "q4" else weight8(g, N, K) for _ in range(2)]
        self.w = [m[2] for m in made]
        self.h = [ctx.register_weight4(m[0], m[1], K, group) if form == "q4" else ctx.register_weight(m[0], m[1]) for m in made]
        self.b = [g.standard_normal(N).astype(np.float32) * np.float32(0.3) if bias else None for _ in range(2)]
        self.call = {"q8": ctx.gated_q8, "q4": ctx.gated_q4, "w8a8": ctx.w8a8_gated}[form]
        self.call_dev = {"q8": ctx.gated_q8_dev, "q4": ctx.gated_q4_dev}.get(form)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for h in self.h:
            (self.ctx.release_weight4 if self.form == "q4" else self.ctx.release_weight)(h)

    def run(self, a, act):
        return self.call(self.h[0], self.h[1], a, self.b[0], self.b[1], ACTS[act])

    def want(self, a, act):
        """(out, bound)"""
        if self.form == "w8a8":
            y = [self.ctx.linear(h, a, bias=b).astype(np.float64) for h, b in zip(self.h, self.b)]
            x = act64(act, y[0])
            return x * y[1], act_bound(act, y[0]) * np.abs(y[1]) + U * np.abs(x * y[1]) + 1e-37
        y = [product(a, w) for w in self.w]
        y = [(v + b, e + U * (np.abs(v) + np.abs(b))) if b is not None else (v, e) for (v, e), b in zip(y, self.b)]
        return gated(*y[0], *y[1], act)


def activations(g, M, K):
    return (g.standard_normal((M, K)) * np.where(g.random((M, K)) < 0.01, 20, 1)).astype(np.float32)


FORMS = ["q8", "q4", "w8a8"]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("N,K", SHAPES)
def test_against_float64(ctx, form, N, K):
    g = np.random.default_rng(N * 7 + K)
    for bias, act in ((True, "silu"), (False, "gelu")):
        with Pair(ctx, form, g, N, K, group=64 if K > 500 else 32, bias=bias) as p:
            for M in MS:
                say(f"gated {form} M={M} N={N} K={K} {act} bias={bias}")
                a = activations(g, M, K)
                got = p.run(a, act)
                want, tol = p.want(a, act)
                assert np.all(np.abs(got - want) <= tol), f"{np.nanmax(np.abs(got - want) / tol)} of the bound"
                assert np.array_equal(got, p.run(a, act))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M,K,N", LARGE)
def test_many_rows(ctx, form, act, M, K, N):
    g = np.random.default_rng(M)
    with Pair(ctx, form, g, N, K, group=128) as p:
        say(f"gated {form} M={M} N={N} K={K} {act}")
        a = activations(g, M, K)
        a[M // 2] = 0
        want, tol = p.want(a, act)
        assert np.all(np.abs(p.run(a, act) - want) <= tol)


@pytest.mark.parametrize("M,K,N", [(20000, 256, 768), (9000, 384, 1500)])
def test_w8a8_whole_batches(ctx, M, K, N):
    # enough rows for the largest tiles, ragged
    g = np.random.default_rng(M)
    for act in ("silu", "gelu"):
        with Pair(ctx, "w8a8", g, N, K) as p:
            say(f"gated w8a8 M={M} N={N} K={K} {act}")
            a = activations(g, M, K)
            want, tol = p.want(a, act)
            assert np.all(np.abs(p.run(a, act) - want) <= tol)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("M", [1, 4, 33, 300])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gate_values(ctx, form, M, act):
    # zero activations: the pre-activations are the biases, any f32
    sp = np.array([0.0, -0.0, 1.0, -1.0, 1e-30, -1e-30, 1e-42, 20.0, -20.0, 80.0, -80.0, 87.0, -87.0, 88.0, -88.0, 89.0, -89.0,
                   100.0, -100.0, 1e30, -1e30, 3e38, -3e38, np.inf, -np.inf, np.nan, 4.0, -4.0, 5.6, -5.6, 1.4142135, -1.4142135])
    rest = np.random.default_rng(9).uniform(-12, 12, size=300)
    x = np.concatenate([sp, rest]).astype(np.float32)
    N = len(x)
    g = np.random.default_rng(2)
    with Pair(ctx, form, g, N, 64) as p:
        p.b = [x, np.full(N, 0.5, np.float32)]
        say(f"gate values {form} M={M} {act}")
        got = p.run(np.zeros((M, 64), np.float32), act).astype(np.float64)
        x64 = x.astype(np.float64)
        want = act64(act, x64) * 0.5
        if act == "gelu":
            ok = np.isfinite(want)  # GELUF32's own limits: 0.5 x (1 + erf)
        else:
            assert np.array_equal(np.isnan(got[0]), np.isnan(want))
            assert got[0][np.isposinf(x64)][0] == np.inf
            ok = np.isfinite(want)
        for row in got:
            assert np.all(np.abs(row[ok] - want[ok]) <= 0.5 * act_bound(act, x64[ok]) + 1e-37)


@pytest.mark.parametrize("form", ["q8", "q4"])
@pytest.mark.parametrize("M", [1, 3, 5, 33, 200, 700])
@pytest.mark.parametrize("K,pad,off", [(768, 4, 0), (100, 3, 1), (33, 0, 0), (1024, 0, 2)])
def test_dev_pitches(ctx, form, M, K, pad, off):
    import torch

    N = 200
    g = np.random.default_rng(K + M)
    with Pair(ctx, form, g, N, K) as p:
        say(f"gated {form} dev M={M} K={K} pad={pad} off={off}")
        a = activations(g, M, K)
        buf = torch.full((M * (K + pad) + off,), float("nan"), device="cuda")
        da = buf[off:].view(M, K + pad)
        da[:, :K] = torch.from_numpy(a).cuda()
        b = [torch.from_numpy(x).cuda() for x in p.b]
        dd = torch.full((M + 2, N + 5), -7.0, device="cuda")
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        p.call_dev(p.h[0], p.h[1], da.data_ptr(), K + pad, M, b[0].data_ptr(), b[1].data_ptr(), enchip.ACT_SILU, dd.data_ptr(),
                   N + 5, stream=st.cuda_stream)
        st.synchronize()
        got = dd.cpu().numpy()
        want, tol = p.want(a, "silu")
        assert np.all(np.abs(got[:M, :N] - want) <= tol)
        assert np.all(got[:, N:] == -7.0) and np.all(got[M:] == -7.0)


@pytest.mark.parametrize("M", [5, 40, 700])
def test_w8a8_dev_streams_share_the_scratch(ctx, M):
    # alternating streams with the linear that shares the scratch, rows behind the last left alone
    import torch

    g = np.random.default_rng(M)
    K, N = 384, 1536
    with Pair(ctx, "w8a8", g, N, K) as p:
        b = [torch.from_numpy(x).cuda() for x in p.b]
        acts = [activations(g, M, K) for _ in range(4)]
        want = [p.run(a, "silu") for a in acts]
        da = [torch.from_numpy(a).cuda() for a in acts]
        out = [torch.full((M + 1, N), -7.0, device="cuda") for _ in acts]
        lin = torch.empty((M, N), device="cuda")
        st = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        say(f"gated w8a8 M={M} on two streams")
        for r in range(3):
            for i, (x, y) in enumerate(zip(da, out)):
                s = st[i % 2].cuda_stream
                ctx.w8a8_gated_dev(p.h[0], p.h[1], x.data_ptr(), M, b[0].data_ptr(), b[1].data_ptr(), enchip.ACT_SILU,
                                   y.data_ptr(), stream=s)
                ctx.linear_dev(p.h[0], x.data_ptr(), M, 0, enchip.ACT_NONE, lin.data_ptr(), stream=st[1].cuda_stream)
        torch.cuda.synchronize()
        for y, w in zip(out, want):
            assert np.array_equal(y[:M].cpu().numpy(), w)
            assert (y[M] == -7.0).all()


@pytest.mark.parametrize("form", FORMS)
def test_same_weight_twice_and_graph(ctx, form):
    import torch

    g = np.random.default_rng(4)
    M, N, K = 24, 300, 256
    with Pair(ctx, form, g, N, K, bias=False) as p:
        a = activations(g, M, K)
        one = p.call(p.h[0], p.h[0], a)  # gate == up
        y = p.call(p.h[0], p.h[1], a)
        s = torch.cuda.Stream()
        da, dd = torch.from_numpy(a).cuda(), torch.empty((M, N), device="cuda")
        torch.cuda.synchronize()

        def run():
            if form == "w8a8":
                ctx.w8a8_gated_dev(p.h[0], p.h[1], da.data_ptr(), M, 0, 0, enchip.ACT_SILU, dd.data_ptr(), stream=s.cuda_stream)
            else:
                p.call_dev(p.h[0], p.h[1], da.data_ptr(), K, M, 0, 0, enchip.ACT_SILU, dd.data_ptr(), N, stream=s.cuda_stream)

        run()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            run()
        for r in range(4):
            x = activations(g, M, K)
            da.copy_(torch.from_numpy(x))
            dd.fill_(-1.0)
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            assert np.array_equal(dd.cpu().numpy(), p.call(p.h[0], p.h[1], x)), r
        del gr
        want, tol = p.want(a, "silu")
        assert np.all(np.abs(y - want) <= tol)
        both, p.w[1], p.h = p.h, p.w[0], [p.h[0], p.h[0]]
        want, tol = p.want(a, "silu")
        p.h = both
        assert np.all(np.abs(one - want) <= tol)


def test_w8a8_row_lengths_in_turn(ctx):
    # one kernel's on-chip memory grows and shrinks from call to call; one launch and codes first
    g = np.random.default_rng(21)
    pairs = [Pair(ctx, "w8a8", g, 96, K) for K in (2048, 1500, 4096, 1100, 3000)]
    wide = Pair(ctx, "w8a8", g, 9000, 64)
    try:
        for M in (1, 8, 20, 32):
            for p in pairs + pairs[::-1] + [wide]:
                a = activations(g, M, p.K)
                want, tol = p.want(a, "silu")
                assert np.all(np.abs(p.run(a, "silu") - want) <= tol), (M, p.K)
    finally:
        for p in pairs + [wide]:
            p.__exit__()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("M", [1, 40])
def test_one_bias(ctx, form, M):
    g = np.random.default_rng(6)
    for which in (0, 1):
        with Pair(ctx, form, g, 90, 100) as p:
            p.b[which] = None
            a = activations(g, M, 100)
            want, tol = p.want(a, "silu")
            assert np.all(np.abs(p.run(a, "silu") - want) <= tol)


@pytest.mark.parametrize("form", FORMS)
def test_captured_call_outlives_larger_ones(form):
    """A graph keeps the scratch it was captured with when a larger call outgrows it."""
    import torch

    with enchip.Context(0) as c:
        g = np.random.default_rng(8)
        M, N, K = 90, 256, 320
        with Pair(c, form, g, N, K) as p:
            s = torch.cuda.Stream()
            acts = [activations(g, m, K) for m in (M, 20 * M)]
            da = [torch.from_numpy(a).cuda() for a in acts]
            dd = [torch.empty((len(a), N), device="cuda") for a in acts]
            b = [torch.from_numpy(x).cuda() for x in p.b]
            torch.cuda.synchronize()

            def run(i):
                if form == "w8a8":
                    c.w8a8_gated_dev(p.h[0], p.h[1], da[i].data_ptr(), len(acts[i]), b[0].data_ptr(), b[1].data_ptr(),
                                     enchip.ACT_SILU, dd[i].data_ptr(), stream=s.cuda_stream)
                else:
                    p.call_dev(p.h[0], p.h[1], da[i].data_ptr(), K, len(acts[i]), b[0].data_ptr(), b[1].data_ptr(),
                               enchip.ACT_SILU, dd[i].data_ptr(), N, stream=s.cuda_stream)

            run(0)
            torch.cuda.synchronize()
            want = dd[0].cpu().numpy()
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=s):
                run(0)
            run(1)
            torch.cuda.synchronize()
            big = dd[1].cpu().numpy()
            filler = torch.full((64 << 20,), float("nan"), device="cuda")  # what freed memory would be given to
            for r in range(3):
                dd[0].zero_()
                torch.cuda.synchronize()
                gr.replay()
                torch.cuda.synchronize()
                assert np.array_equal(dd[0].cpu().numpy(), want), r
                run(1)
                torch.cuda.synchronize()
                assert np.array_equal(dd[1].cpu().numpy(), big), r
            del gr, filler


def test_threads_share_a_context(ctx):
    from concurrent.futures import ThreadPoolExecutor

    g = np.random.default_rng(12)
    pairs = {f: Pair(ctx, f, g, 300, 256) for f in FORMS}
    try:
        jobs = [(f, activations(g, M, 256)) for f in FORMS for M in (1, 30, 200, 1000)]
        want = [pairs[f].run(a, "silu") for f, a in jobs]
        with ThreadPoolExecutor(8) as ex:
            for _ in range(3):
                got = list(ex.map(lambda j: pairs[j[0]].run(j[1], "silu"), jobs))
                assert all(np.array_equal(x, y) for x, y in zip(got, want))
    finally:
        for p in pairs.values():
            p.__exit__()


def test_refusals(ctx):
    import torch

    g = np.random.default_rng(1)
    mk = lambda N, K: ctx.register_weight(*weight8(g, N, K)[:2])  # noqa: E731
    mk4 = lambda N, K, gr: ctx.register_weight4(*weight4(g, N, K, gr)[:2], K, gr)  # noqa: E731
    a, b, c, inf = mk(40, 64), mk(40, 96), mk(48, 64), ctx.register_weight(np.ones((40, 64), np.int8), np.full(40, np.inf, np.float32))
    k0 = ctx.register_weight(np.zeros((40, 0), np.int8), np.ones(40, np.float32))
    a4, b4 = mk4(40, 64, 32), mk4(40, 64, 64)
    d = torch.zeros(8192, device="cuda")
    p = d.data_ptr()

    def refused(call, *args, code=enchip.ERR_ARG):
        with pytest.raises(enchip.EnchipError) as e:
            call(*args)
        assert e.value.code == code, args

    S = enchip.ACT_SILU
    for gate, up in ((a, b), (a, c), (k0, k0)):
        refused(ctx.gated_q8_dev, gate, up, p, 96, 2, 0, 0, S, p, 48)
        refused(ctx.w8a8_gated_dev, gate, up, p, 2, 0, 0, S, p)
    refused(ctx.gated_q8_dev, a, inf, p, 64, 2, 0, 0, S, p, 40)
    refused(ctx.gated_q8_dev, inf, a, p, 64, 2, 0, 0, S, p, 40)
    refused(ctx.gated_q4_dev, a4, b4, p, 64, 2, 0, 0, S, p, 40)
    refused(ctx.gated_q4_dev, a4, a, p, 64, 2, 0, 0, S, p, 40, code=enchip.ERR_HANDLE)
    refused(ctx.gated_q8_dev, a, a4, p, 64, 2, 0, 0, S, p, 40, code=enchip.ERR_HANDLE)
    for act in (enchip.ACT_NONE, enchip.ACT_TANH, 7, -1):
        refused(ctx.gated_q8_dev, a, a, p, 64, 2, 0, 0, act, p, 40)
        refused(ctx.gated_q4_dev, a4, a4, p, 64, 2, 0, 0, act, p, 40)
        refused(ctx.w8a8_gated_dev, a, a, p, 2, 0, 0, act, p)
    for call, w in ((ctx.gated_q8_dev, a), (ctx.gated_q4_dev, a4)):
        for args in ((p, 63, 2, 0, 0, S, p, 40), (p, 64, 2, 0, 0, S, p, 39), (0, 64, 2, 0, 0, S, p, 40), (p, 64, 2, 0, 0, S, 0, 40),
                     (p, 64, -1, 0, 0, S, p, 40), (p, 64, 1 << 32, 0, 0, S, p, 40)):
            refused(call, w, w, *args)
        call(w, w, 0, 64, 0, 0, 0, S, 0, 40)  # no rows: nothing to do
    refused(ctx.w8a8_gated_dev, a, a, 0, 2, 0, 0, S, p)
    refused(ctx.w8a8_gated_dev, a, a, p, 2, 0, 0, S, 0)
    refused(ctx.w8a8_gated_dev, a, a, p, -1, 0, 0, S, p)
    ctx.w8a8_gated_dev(a, a, 0, 0, 0, 0, S, 0)
    for act in (enchip.ACT_NONE, enchip.ACT_TANH):  # the gates' own activation is no other call's
        refused(ctx.w8a8_gated, a, a, np.zeros((1, 64), np.float32), None, None, act)
    refused(ctx.linear_dev, a, p, 1, 0, S, p)
    refused(ctx.bias_act_rows_dev, p, 8, 1, 8, 0, S)
    with pytest.raises(ValueError):
        ctx.gated_q8(a, a, np.zeros((2, 63), np.float32))
    with pytest.raises(ValueError):
        ctx.gated_q8(a, a, np.zeros((2, 64), np.float32), bias_up=np.zeros(39, np.float32))
    for w in (a, b, c, inf, k0):
        ctx.release_weight(w)
    for w in (a4, b4):
        ctx.release_weight4(w)
    refused(ctx.gated_q8_dev, a, a, p, 64, 2, 0, 0, S, p, 40, code=enchip.ERR_HANDLE)
