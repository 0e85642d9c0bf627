"""Attention with a relative position bias over spans (enchip_attention_bias_dev) against float64.

The tolerance per element. Products are within 3 2^-22 of exact and sums of hd f32 terms round hd times, so a score
is off by at most delta = scale (hd 2^-24 + 3 2^-22) sum |q k| + 2^-22 |y| (its f32 value and the bias in base 2), with
the parts' 2^-25 floor another scale hd 2^-24 (max|q| + max|k|). Weights and their sum are off by twice that,
2^-21 of 2^x, and 3 2^-22 of the second product, and the sums over n keys round n times (and once a tile for the
running maximum): (2 delta + (n + 64) 2^-24) max|v| in all, and 2^-24 for v's floor."""
import numpy as np
import pytest

from aikit_amd import enchip
from block_oracle import attention, bucket_of

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


class Case:
    def __init__(self, heads, kv, hd, T, seed=0, std=1.0, pad=0, table=None, reach=20, buckets=16):
        g = np.random.default_rng(seed + T * 7 + heads)
        self.heads, self.kv, self.hd, self.T = heads, kv, hd, T
        self.ld = (heads + 2 * kv) * hd + pad
        self.x = (g.standard_normal((T, self.ld)) * std).astype(np.float32)
        self.table = g.standard_normal((buckets, heads)).astype(np.float32) if table is None else table
        self.reach = reach
        self.scale = hd ** -0.5

    def parts(self):
        a, b = self.heads * self.hd, (self.heads + self.kv) * self.hd
        return (self.x[:, s].astype(np.float64) for s in (slice(0, a), slice(a, b), slice(b, b + self.kv * self.hd)))

    def run(self, ctx, spans=None, nseq=None, L=None, bias="log", ldo=None, off=0, fill=3.0, stream=0, scale=None, rp=None):
        import torch

        W = self.heads * self.hd
        ldo = W if ldo is None else ldo
        d = torch.from_numpy(self.x).cuda()
        out = torch.full((off + self.T * ldo + 4,), fill, device="cuda")
        own = rp is None and bias is not None
        if own:
            rp = ctx.relpos(self.table, self.reach)
        sp = None if spans is None else torch.tensor(spans, dtype=torch.int32, device="cuda").reshape(-1, 2).contiguous()
        p = d.data_ptr()
        try:
            torch.cuda.synchronize()
            ctx.attention_bias_dev(rp, p, self.ld, p + 4 * W, self.ld, p + 4 * (W + self.kv * self.hd), self.ld,
                                   out.data_ptr() + 4 * off, ldo, len(spans) if spans is not None else nseq,
                                   self.T if spans is not None else L, self.heads, self.kv, self.hd,
                                   self.scale if scale is None else scale, 0 if sp is None else sp.data_ptr(), stream)
            torch.cuda.synchronize()
        finally:
            if own:
                ctx.release_relpos(rp)
        got = out.cpu().numpy()
        body = got[off:off + self.T * ldo].reshape(self.T, ldo)
        assert (got[:off] == fill).all() and (got[off + self.T * ldo:] == fill).all() and (body[:, W:] == fill).all()
        return body[:, :W]

    def check(self, ctx, spans=None, nseq=None, L=None, bias="log", scale=None, rp=None, fn=None, **k):
        fill = k.get("fill", 3.0)
        got = self.run(ctx, spans, nseq, L, bias, scale=scale, rp=rp, **k)
        rows = spans if spans is not None else [(z * L, (z + 1) * L) for z in range(nseq)]
        q, kk, v = self.parts()
        s = self.scale if scale is None else scale
        nb = len(self.table)
        if fn is None and bias is not None:
            def fn(d, h):
                return self.table[bucket_of(d, nb, self.reach), h].astype(np.float64)
        want = attention(q, kk, v, rows, self.heads, self.kv, self.hd, s, fn, np.full((self.T, self.heads * self.hd), fill))
        tol = np.zeros_like(want)
        for a, b in rows:
            if b <= a:
                continue
            hs, G = self.hd, self.heads // self.kv
            for h in range(self.heads):
                c, cg = slice(h * hs, (h + 1) * hs), slice((h // G) * hs, (h // G + 1) * hs)
                mass = np.abs(q[a:b, c]) @ np.abs(kk[a:b, cg]).T
                top = np.abs(self.table[np.isfinite(self.table)]).max(initial=0) if bias is not None or fn is not None else 0
                floor = hs * 2.0 ** -24 * (np.abs(q[a:b, c]).max() + np.abs(kk[a:b, cg]).max())
                delta = abs(s) * ((hs * 2.0 ** -24 + 3 * 2.0 ** -22) * mass.max(axis=1, keepdims=True) + floor) + \
                    2.0 ** -22 * (abs(s) * mass.max(axis=1, keepdims=True) + top)
                tol[a:b, c] = (2 * delta + (b - a + 64) * 2.0 ** -24) * np.abs(v[a:b, cg]).max() + 2.0 ** -24
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], tol[bad][:3])
        # the rows' errors are rounding, not a bound's worst case: as a whole 2-norm 2^-17
        num, den = np.linalg.norm(got - want), np.linalg.norm(want)
        assert num <= 2.0 ** -17 * den, num / den


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("nseq,L", [(1, 1), (3, 2), (2, 31), (1, 33), (2, 64), (1, 65), (1, 129), (1, 256), (1, 257), (2, 300), (1, 513), (1, 1030)])
def test_lengths(ctx, hd, nseq, L):
    say(f"attention_bias hd={hd} nseq={nseq} L={L}")
    Case(3, 3, hd, nseq * L).check(ctx, nseq=nseq, L=L)


@pytest.mark.parametrize("heads,kv,hd", [(4, 1, 64), (6, 2, 32), (8, 4, 128), (1, 1, 64), (5, 5, 64)])
def test_grouped_heads(ctx, heads, kv, hd):
    say(f"attention_bias heads={heads} kv={kv} hd={hd}")
    Case(heads, kv, hd, 2 * 70).check(ctx, nseq=2, L=70)


SPANS = {
    "padded": ([(0, 40), (40, 40), (80, 81), (120, 160)], 160),
    "packed": ([(0, 1), (1, 4), (4, 130), (130, 130), (130, 500), (500, 501)], 501),
    "gaps": ([(3, 9), (9, 9), (20, 21), (50, 320), (400, 430)], 437),
    "one": ([(5, 6)], 40),
    "whole": ([(0, 333)], 333),
    "empty": ([(7, 7), (7, 7)], 20),
    "many": ([(3 * i, 3 * i + (i % 4 > 0) * 2) for i in range(300)], 900),
    "past the end": ([(0, 10), (90, 2000)], 100),
    "backwards": ([(10, 5), (20, 30)], 64),
}


@pytest.mark.parametrize("name", sorted(SPANS))
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_spans(ctx, name, hd):
    spans, T = SPANS[name]
    say(f"attention_bias spans {name} hd={hd}")
    cut = [(max(a, 0), min(b, T)) for a, b in spans]
    c = Case(4, 2, hd, T)
    # rows of no span hold infinities and NaN: nothing reads them
    inside = np.zeros(T, bool)
    for a, b in cut:
        inside[a:b] = True
    c.x[~inside] = np.where(np.arange(c.ld) % 2 == 0, np.nan, np.inf)
    got = c.run(ctx, spans=spans)
    assert (got[~inside] == 3.0).all()
    c.x[~inside] = 0
    if name in ("past the end", "backwards"):
        c2 = Case(4, 2, hd, T)
        c2.x = c.x
        q, k, v = c2.parts()
        want = attention(q, k, v, cut, 4, 2, hd, c2.scale, lambda d, h: c2.table[bucket_of(d, 16, 20), h].astype(np.float64),
                         np.full((T, 4 * hd), 3.0))
        assert np.abs(got - want).max() <= 2e-4
    else:
        c.check(ctx, spans=spans)


def test_spans_out_of_order_stay_in_bounds(ctx):
    # not a valid call: rows may stay as they were, and nothing outside the buffers is touched
    say("attention_bias spans out of order")
    c = Case(2, 2, 64, 300)
    got = c.run(ctx, spans=[(200, 300), (0, 100), (100, 150), (-50, 20), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, 2 ** 31 - 1)])
    assert np.isfinite(got).all()


@pytest.mark.parametrize("hd,heads,kv,nseq,L", [
    # every form of the kernel by its sizes: a wavefront alone, tiles of 256 and 512 queries, keys in parts
    (32, 12, 12, 70, 33), (64, 12, 12, 70, 33), (128, 12, 12, 70, 33), (128, 12, 3, 70, 33),
    (32, 8, 8, 16, 300), (64, 8, 8, 16, 300), (128, 8, 8, 16, 300), (64, 12, 4, 43, 512), (64, 16, 16, 16, 512),
    (32, 3, 3, 1, 1500), (64, 3, 3, 1, 1500), (128, 3, 3, 1, 1500), (64, 2, 1, 1, 3000), (32, 1, 1, 1, 4099), (64, 1, 1, 2, 2111),
    (128, 4, 1, 1, 1300),
])
def test_forms(ctx, hd, heads, kv, nseq, L):
    say(f"attention_bias form hd={hd} heads={heads} kv={kv} {nseq}x{L}")
    Case(heads, kv, hd, nseq * L).check(ctx, nseq=nseq, L=L)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_parts_of_spans(ctx, hd):
    # a mean length that splits keys, lengths that leave parts empty, rows between the spans
    say(f"attention_bias parts of spans hd={hd}")
    spans = [(0, 2000), (2000, 2001), (2050, 3300), (3300, 3300), (3301, 6000)]
    Case(2, 1, hd, 6100).check(ctx, spans=spans, ldo=2 * hd + 3)


def test_no_bias_and_scales(ctx):
    say("attention_bias without a bias; scales of either sign and 0")
    for scale in (0.125, -0.2, 0.0):
        Case(3, 3, 64, 2 * 90).check(ctx, nseq=2, L=90, bias=None, scale=scale)
        Case(3, 3, 64, 2 * 90).check(ctx, nseq=2, L=90, scale=scale)


@pytest.mark.parametrize("buckets,reach", [(4, 2), (8, 5), (16, 64), (32, 128), (64, 1000), (32, 9)])
def test_buckets(ctx, buckets, reach):
    say(f"attention_bias buckets={buckets} reach={reach}")
    Case(2, 2, 32, 300, buckets=buckets, reach=reach).check(ctx, nseq=1, L=300)


def test_bucket_map(ctx):
    say("attention_bias buckets by a map; windows by -infinity; rows that attend to nothing")
    g = np.random.default_rng(3)
    table = g.standard_normal((7, 2)).astype(np.float32)
    table[6] = -np.inf
    reach = 11
    m = g.integers(0, 6, 2 * reach + 1)
    m[0] = m[-1] = 6  # a window of 10 rows each way
    c = Case(2, 2, 64, 150, table=table)
    fn = lambda d, h: table[m[np.clip(d, -reach, reach) + reach], h].astype(np.float64)  # noqa: E731
    rp = ctx.relpos_from_map(table, m)
    try:
        c.check(ctx, nseq=1, L=150, rp=rp, fn=fn)
        c.check(ctx, spans=[(0, 3), (3, 150)], rp=rp, fn=fn)
    finally:
        ctx.release_relpos(rp)
    # keys before the query only, the query's own row not among them: the first row attends to nothing
    m = np.where(np.arange(-1, 2) < 0, 0, 6)
    rp = ctx.relpos_from_map(table, m)
    try:
        fn = lambda d, h: table[m[np.clip(d, -1, 1) + 1], h].astype(np.float64)  # noqa: E731
        got = c.run(ctx, nseq=1, L=150, rp=rp)
        assert (got[0] == 0).all()
        c.check(ctx, nseq=1, L=150, rp=rp, fn=fn)
        # one bucket for every distance, all of it -infinity: zeros
        z = ctx.relpos_from_map(np.full((1, 2), -np.inf, np.float32), np.zeros(1, np.int32))
        try:
            assert (c.run(ctx, nseq=1, L=150, rp=z) == 0).all()
        finally:
            ctx.release_relpos(z)
    finally:
        ctx.release_relpos(rp)


def test_large_biases(ctx):
    say("attention_bias biases of 2^100 and -2^100")
    table = np.array([[2.0 ** 100, -2.0 ** 100], [2.0 ** 100, -2.0 ** 100]], np.float32)
    c = Case(2, 2, 32, 77, table=table)
    rp = ctx.relpos_from_map(table, np.array([0, 1, 0], np.int32))
    try:  # scores vanish beside the bias: every key weighs the same
        got = c.run(ctx, nseq=1, L=77, rp=rp)
        _, _, v = c.parts()
        assert np.abs(got - v.mean(axis=0)).max() <= 77 * 2.0 ** -22 * np.abs(v).max()
    finally:
        ctx.release_relpos(rp)


def test_pitches_and_alignment(ctx):
    say("attention_bias pitches, an output that is not aligned")
    c = Case(3, 3, 64, 140, pad=12)
    c.check(ctx, nseq=2, L=70, ldo=3 * 64 + 5)
    c.check(ctx, nseq=2, L=70, ldo=3 * 64 + 8, off=1)


def test_wide_scores(ctx):
    # standard deviation 4: scores of +-100, weights on one key
    say("attention_bias wide scores")
    Case(2, 2, 64, 200, std=4.0).check(ctx, nseq=1, L=200)


def test_infinite_and_nan_keys(ctx):
    say("attention_bias infinities and NaN within a span")
    c = Case(2, 2, 64, 120)
    c.x[30, 2 * 64 + 5] = np.nan          # head 0's key 30
    c.x[90, 4 * 64 + 64 + 1] = np.inf     # head 1's value 90
    got = c.run(ctx, spans=[(0, 60), (60, 120)])
    assert np.isnan(got[:60, :64]).all() and np.isfinite(got[60:, :64]).all()
    assert np.isfinite(got[:60, 64:]).all() and np.isnan(got[60:, 65]).all()


def test_more_blocks_than_one_round(ctx):
    # many sequences of many lengths: every one against the same rows called alone
    import torch

    say("attention_bias 500 packed sequences against single calls")
    g = np.random.default_rng(9)
    n = g.integers(0, 40, 500)
    n[::50] = 300
    at = np.concatenate([[0], np.cumsum(n)])
    spans = [(int(a), int(b)) for a, b in zip(at[:-1], at[1:])]
    c = Case(2, 1, 64, int(at[-1]))
    got = c.run(ctx, spans=spans)
    for z in (0, 1, 49, 50, 51, 250, 499):
        a, b = spans[z]
        if b > a:
            one = Case(2, 1, 64, b - a)
            one.x, one.table = c.x[a:b].copy(), c.table
            # the kernel, and with it the order of the sums, goes by the sizes: each is within 2^-17 of the formula in
            # all (Case.check), so they are within 2^-16 of each other
            alone = one.run(ctx, nseq=1, L=b - a)
            assert np.linalg.norm(alone - got[a:b]) <= 2.0 ** -16 * np.linalg.norm(alone)
            one.check(ctx, nseq=1, L=b - a)
    torch.cuda.synchronize()


def test_streams_and_graph(ctx):
    import torch

    s = torch.cuda.Stream()
    heads, kv, hd, T = 4, 2, 64, 500
    W = (heads + 2 * kv) * hd
    x, y, e = torch.empty((T, W), device="cuda"), *(torch.zeros((T, heads * hd), device="cuda") for _ in range(2))
    spans = torch.tensor([[0, 100], [100, 101], [130, 480]], dtype=torch.int32, device="cuda")
    rp = ctx.relpos(np.random.default_rng(1).standard_normal((32, heads)).astype(np.float32), 128)
    torch.cuda.synchronize()

    def call(out):
        p = x.data_ptr()
        ctx.attention_bias_dev(rp, p, W, p + 4 * heads * hd, W, p + 4 * (heads + kv) * hd, W, out.data_ptr(), heads * hd, 3, T, heads,
                               kv, hd, 0.125, spans.data_ptr(), s.cuda_stream)

    try:
        with torch.cuda.stream(s):
            x.normal_()
        call(e)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            call(y)
        say("attention_bias captured, 3 replays with other spans")
        for i in range(3):
            with torch.cuda.stream(s):
                x.normal_()
                spans[1, 1] = 101 + 9 * i
                y.zero_(), e.zero_()
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            call(e)
            torch.cuda.synchronize()
            assert torch.equal(y, e)
        del gr
    finally:
        ctx.release_relpos(rp)


def test_parts_in_a_graph_and_on_two_streams(ctx):
    import torch

    heads, hd, T = 2, 64, 2500
    W = 3 * heads * hd
    x = torch.empty((T, W), device="cuda")
    y, e, z = (torch.zeros((T, heads * hd), device="cuda") for _ in range(3))
    rp = ctx.relpos(np.random.default_rng(2).standard_normal((32, heads)).astype(np.float32), 128)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def call(out, stream):
        p = x.data_ptr()
        ctx.attention_bias_dev(rp, p, W, p + 4 * heads * hd, W, p + 8 * heads * hd, W, out.data_ptr(), heads * hd, 1, T, heads, heads, hd,
                               0.125, stream=stream)

    try:
        with torch.cuda.stream(s):
            x.normal_()
        call(e, s.cuda_stream)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            call(y, s.cuda_stream)
        say("attention_bias in parts captured, 3 replays; two streams on the shared scratch")
        for _ in range(3):
            with torch.cuda.stream(s):
                x.normal_()
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            call(e, s.cuda_stream)
            torch.cuda.synchronize()
            assert torch.equal(y, e)
        del gr
        for _ in range(6):
            call(y, s.cuda_stream), call(z, t.cuda_stream), call(e, 0)
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.equal(y, e)
        ctx.set_scratch_limit(1000)
        try:
            with pytest.raises(enchip.EnchipError) as err:
                call(y, 0)
            assert err.value.code == enchip.ERR_OOM
        finally:
            ctx.set_scratch_limit(0)
    finally:
        ctx.release_relpos(rp)


def test_refusals(ctx):
    import torch

    x = torch.zeros(1 << 16, device="cuda")
    p, o = x.data_ptr(), x.data_ptr() + 4 * 32768
    sp = torch.tensor([[0, 2], [2, 4]], dtype=torch.int32, device="cuda")
    rp = ctx.relpos(np.zeros((8, 4), np.float32), 20)

    def call(b=rp, q=p, ldq=256, k=p, ldk=256, v=p, ldv=256, out=o, ldo=256, nseq=2, L=4, heads=4, kv=4, hd=64, spans=0):
        ctx.attention_bias_dev(b, q, ldq, k, ldk, v, ldv, out, ldo, nseq, L, heads, kv, hd, 1.0, spans)

    try:
        call(), call(spans=sp.data_ptr()), call(b=None), call(nseq=0), call(L=0), call(b=None, heads=0, kv=0), call(kv=2), call(ldo=257)
        for k in (dict(hd=48), dict(hd=256), dict(kv=3), dict(kv=0), dict(kv=8), dict(heads=-1), dict(nseq=-1), dict(L=-1), dict(ldq=252),
                  dict(ldq=258), dict(ldk=254), dict(ldv=255), dict(ldk=192), dict(ldo=255), dict(q=0), dict(k=0), dict(v=0), dict(out=0),
                  dict(q=p + 4), dict(k=p + 8), dict(v=p + 4), dict(spans=sp.data_ptr() + 4), dict(heads=2, kv=2), dict(L=2 ** 31),
                  dict(nseq=2 ** 22, L=1024), dict(nseq=2 ** 23, spans=sp.data_ptr()), dict(ldq=2 ** 25), dict(ldk=2 ** 25),
                  dict(heads=65536, kv=65536, ldq=2 ** 22, ldk=2 ** 22, ldv=2 ** 22, ldo=2 ** 22, b=None)):
            with pytest.raises(enchip.EnchipError) as err:
                call(**k)
            assert err.value.code == enchip.ERR_ARG, k
        with pytest.raises(enchip.EnchipError) as err:
            call(b=enchip.RelPos(10 ** 9, 4))
        assert err.value.code == enchip.ERR_HANDLE
        f = lambda *s: np.zeros(s, np.float32)  # noqa: E731
        for t, d in ((f(7, 2), 20), (f(2, 2), 20), (f(8, 2), 2), (f(8, 0), 20), (f(0, 2), 20), (f(8, 2), 2 ** 21),
                     (np.full((8, 2), np.nan, np.float32), 20), (np.full((8, 2), np.inf, np.float32), 20),
                     (np.full((8, 2), np.finfo(np.float32).min, np.float32), 20), (np.full((8, 2), 2.0 ** 101, np.float32), 20),
                     (f(8, 60000), 2 ** 20)):
            with pytest.raises(enchip.EnchipError) as err:
                ctx.relpos(t, d)
            assert err.value.code == enchip.ERR_ARG
        for m in ([0, 8, 0], [0, -1, 0]):
            with pytest.raises(enchip.EnchipError):
                ctx.relpos_from_map(f(8, 2), np.array(m, np.int32))
        with pytest.raises(enchip.EnchipError) as err:
            ctx.release_relpos(enchip.RelPos(10 ** 9, 4))
        assert err.value.code == enchip.ERR_HANDLE
        torch.cuda.synchronize()
    finally:
        ctx.release_relpos(rp)


def test_pool_spans(ctx):
    import torch

    say("pool_mean_l2_spans against pool_mean_l2 of each span")
    g = np.random.default_rng(4)
    h = torch.from_numpy(g.standard_normal((400, 96)).astype(np.float32)).cuda()
    spans = [(0, 1), (1, 1), (1, 130), (350, 400), (140, 141), (390, 5000), (-20, 3)]
    sp = torch.tensor(spans, dtype=torch.int32, device="cuda")
    out = torch.full((len(spans), 96), 9.0, device="cuda")
    torch.cuda.synchronize()
    ctx.pool_mean_l2_spans_dev(h.data_ptr(), 96, 400, sp.data_ptr(), len(spans), 96, out.data_ptr(), 96)
    for i, (a, b) in enumerate(spans):
        a, b = max(a, 0), min(b, 400)
        one = torch.full((1, 96), 9.0, device="cuda")
        torch.cuda.synchronize()
        ctx.pool_mean_l2_dev(h[a:b].contiguous().data_ptr() if b > a else h.data_ptr(), 96, 1, b - a, 96, one.data_ptr(), 96)
        torch.cuda.synchronize()
        assert torch.equal(one[0], out[i]), i
    for k in (dict(spans=0), dict(spans=sp.data_ptr() + 4), dict(nseq=65536), dict(ld=95)):
        with pytest.raises(enchip.EnchipError):
            ctx.pool_mean_l2_spans_dev(h.data_ptr(), k.get("ld", 96), 400, k.get("spans", sp.data_ptr()), k.get("nseq", 7), 96,
                                       out.data_ptr(), 96)
    torch.cuda.synchronize()


def ragged(T, n, seed):
    """n ascending spans of T rows: some empty, some of a row or two, one long, gaps."""
    g = np.random.default_rng(seed)
    size = g.lognormal(0, 1.2, n)
    size[g.random(n) < 0.1] = 0
    size[n // 3] = size.sum() * 0.3
    size = np.floor(size / size.sum() * T * 0.9).astype(int)
    spans, at = [], 0
    for z in size:
        at += int(g.integers(0, 2)) * int(g.integers(0, T // n // 10))
        spans.append((at, min(at + int(z), T)))
        at = spans[-1][1]
    return spans


@pytest.mark.parametrize("heads,kv,hd,T,n", [(32, 32, 32, 3000, 30), (16, 16, 64, 5000, 40), (64, 16, 64, 2600, 33), (16, 2, 64, 9000, 70),
                                             (32, 8, 128, 3000, 30), (10, 10, 128, 5000, 55),
                                             # a wavefront alone: means of 33 to 64 rows
                                             (16, 4, 32, 3700, 110), (24, 24, 64, 3000, 60), (12, 12, 128, 5100, 90)])
@pytest.mark.parametrize("ldo", [0, 3])
def test_longest_first(ctx, heads, kv, hd, T, n, ldo):
    say(f"attention_bias spans longest first heads={heads} kv={kv} hd={hd} T={T} n={n} ldo+{ldo}")
    spans = ragged(T, n, T + n + hd)
    c = Case(heads, kv, hd, T, reach=100, buckets=32)
    inside = np.zeros(T, bool)
    for a, b in spans:
        inside[a:b] = True
    assert not inside.all()
    c.x[~inside] = np.nan
    q = c.x[inside]
    assert np.isfinite(q).all()
    c.check(ctx, spans=spans, ldo=heads * hd + ldo)


def test_longest_first_in_a_graph_and_on_two_streams(ctx):
    import torch

    heads, hd, T, n = 24, 64, 4000, 40
    W = 3 * heads * hd
    x = torch.empty((T, W), device="cuda")
    y, e, z = (torch.zeros((T, heads * hd), device="cuda") for _ in range(3))
    lists = [torch.tensor(ragged(T, n, i), dtype=torch.int32, device="cuda") for i in range(4)]
    spans = lists[3].clone()
    rp = ctx.relpos(np.random.default_rng(2).standard_normal((32, heads)).astype(np.float32), 128)
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def call(out, stream):
        p = x.data_ptr()
        ctx.attention_bias_dev(rp, p, W, p + 4 * heads * hd, W, p + 8 * heads * hd, W, out.data_ptr(), heads * hd, n, T, heads, heads, hd,
                               0.125, spans.data_ptr(), stream)

    try:
        with torch.cuda.stream(s):
            x.normal_()
        call(e, s.cuda_stream)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            call(y, s.cuda_stream)
        say("attention_bias longest first captured, 3 replays with other spans; two streams on the shared scratch")
        for i in range(3):
            with torch.cuda.stream(s):
                x.normal_()
                spans.copy_(lists[i])
                y.zero_(), e.zero_()
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            call(e, s.cuda_stream)
            torch.cuda.synchronize()
            assert torch.equal(y, e)
        del gr
        for u in (y, z, e):
            u.zero_()
        torch.cuda.synchronize()
        for _ in range(6):
            call(y, s.cuda_stream), call(z, t.cuda_stream), call(e, 0)
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.equal(y, e)
    finally:
        ctx.release_relpos(rp)


def test_many_spans_out_of_order_stay_in_bounds(ctx):
    # not a valid call: rows may stay as they were or be another span's, and nothing outside the buffers is touched
    say("attention_bias many spans out of order")
    c = Case(24, 24, 64, 3000)
    far = [(-2 ** 31, 2 ** 31 - 1)] * 10 + [(2900 - 100 * i, 3000 - 100 * i) for i in range(29)] + [(2 ** 31 - 1, -2 ** 31)]
    assert np.isfinite(c.run(ctx, spans=far)).all()
