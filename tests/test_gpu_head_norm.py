"""RMS norms of query and key heads with rotation (enchip_head_norm_rope_rows_dev) against float64.

The tolerance per element. 1 / sqrt is taken in 64 bits and rounded once, applied by two products (the factor,
the gain) that round once each: n is within 3 2^-24 |n|, under 2^-22 |n|. A turned element has in units of
2^-23 m (|n1| + |n2|): 1.5 of n, 0.8 of the reduced angle's rounding (pi 2^-25), 1 of sine and cosine (2 ulp), 0.5
of mscale, 1 of the products and their sum: 4.8, under 5."""
import numpy as np
import pytest

from aikit_amd import enchip
from block_oracle import freqs64, head_norm_rope

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


def run(ctx, qh, kh, hd, rot, layout, nseq, L, pos=None, pos0=0, pad=0, off=0, inplace=False, eps=1e-6, x=None, freqs=None,
        mscale=1.0, stream=None):
    """(outputs, oracle, tolerance, what lay around) of one call; x [rows, (qh + kh) hd] float32 or drawn."""
    import torch

    rows, W = nseq * L, (qh + kh) * hd
    g = np.random.default_rng(rows * 31 + W + rot)
    if x is None:
        x = g.standard_normal((rows, W)).astype(np.float32) * np.exp(g.standard_normal((rows, 1))).astype(np.float32)
    gq, gk = (1 + 0.2 * g.standard_normal((2, hd))).astype(np.float32)
    ld = W + pad
    buf = torch.full((off + rows * ld + 4,), 7.0, device="cuda")
    buf[off:off + rows * ld].view(rows, ld)[:, :W] = torch.from_numpy(x).cuda()
    before = buf.cpu().numpy().copy()
    out = buf if inplace else torch.full((off + rows * ld + 4,), 5.0, device="cuda")
    dq, dk = torch.from_numpy(gq).cuda(), torch.from_numpy(gk).cuda()
    dp = None if pos is None else torch.from_numpy(pos.astype(np.int32)).cuda()
    r = None
    if rot:
        r = ctx.rope_from_freqs(freqs64(rot) if freqs is None else freqs, mscale)
    try:
        torch.cuda.synchronize()
        ctx.head_norm_rope_rows_dev(r, layout, buf.data_ptr() + 4 * off, ld, out.data_ptr() + 4 * off, ld, nseq, L, qh, kh, hd,
                                    dq.data_ptr(), dk.data_ptr(), eps, 0 if dp is None else dp.data_ptr(), pos0,
                                    0 if stream is None else stream)
        torch.cuda.synchronize()
    finally:
        if r is not None:
            ctx.release_rope(r)
    at = pos if pos is not None else pos0 + np.arange(rows) % max(L, 1)
    y, n = head_norm_rope(x.astype(np.float64), qh, kh, hd, gq, gk, eps, at, rot, layout == enchip.ROPE_INTERLEAVED, freqs, mscale)
    tol = np.abs(n) * 2.0 ** -22
    if rot:
        j = np.arange(rot // 2)
        i, k = (2 * j, 2 * j + 1) if layout == enchip.ROPE_INTERLEAVED else (j, j + rot // 2)
        t = 5 * 2.0 ** -23 * abs(mscale) * (np.abs(n[..., i]) + np.abs(n[..., k]))
        tol[..., i] = tol[..., k] = t
    got = out.cpu().numpy()
    body = got[off:off + rows * ld].reshape(rows, ld)
    mark = before if inplace else np.full_like(got, 5.0)
    assert np.array_equal(got[:off], mark[:off]) and np.array_equal(got[off + rows * ld:], mark[off + rows * ld:])
    assert np.array_equal(body[:, W:], mark[off:off + rows * ld].reshape(rows, ld)[:, W:])
    return body[:, :W], y, tol.reshape(rows, W) + 1e-40


def check(ctx, *a, **k):
    got, y, tol = run(ctx, *a, **k)
    bad = np.abs(got.astype(np.float64) - y) > tol
    assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], y[bad][:3])


@pytest.mark.parametrize("qh,kh,hd,rot,layout,nseq,L,k", [
    (12, 12, 32, 32, enchip.ROPE_HALF, 1, 16, {}),
    (12, 12, 64, 64, enchip.ROPE_HALF, 3, 65, {}),
    (16, 4, 128, 64, enchip.ROPE_INTERLEAVED, 1, 301, {}),
    (1, 0, 32, 32, enchip.ROPE_HALF, 1, 1, {}),
    (0, 3, 64, 32, enchip.ROPE_INTERLEAVED, 2, 5, {}),
    (5, 2, 64, 0, enchip.ROPE_HALF, 2, 33, {}),                       # norms alone
    (3, 1, 64, 42, enchip.ROPE_HALF, 1, 19, {}),                      # 21 pairs: single floats
    (3, 1, 64, 42, enchip.ROPE_INTERLEAVED, 1, 19, {}),
    (3, 1, 64, 44, enchip.ROPE_HALF, 1, 19, {}),                      # two floats, a rest of 20
    (2, 1, 33, 20, enchip.ROPE_HALF, 2, 7, {}),                       # an odd head
    (2, 1, 35, 34, enchip.ROPE_INTERLEAVED, 2, 7, {}),                # a rest of one
    (2, 2, 1, 0, enchip.ROPE_HALF, 3, 5, {}),                         # heads of one element
    (2, 1, 2, 2, enchip.ROPE_INTERLEAVED, 3, 5, {}),
    (1, 1, 1024, 1024, enchip.ROPE_HALF, 1, 9, {}),
    (1, 1, 1024, 512, enchip.ROPE_INTERLEAVED, 1, 9, {}),
    (1, 1, 1022, 1022, enchip.ROPE_HALF, 1, 3, {}),                   # 511 slots of single floats
    (1, 1, 514, 514, enchip.ROPE_HALF, 1, 3, {}),
    (1, 2, 770, 512, enchip.ROPE_HALF, 1, 3, {}),
    (1, 1, 1000, 1000, enchip.ROPE_HALF, 1, 3, {}),
    (12, 12, 64, 64, enchip.ROPE_HALF, 1, 50, dict(pad=3)),           # a pitch that is a multiple of nothing
    (12, 12, 64, 64, enchip.ROPE_INTERLEAVED, 1, 50, dict(pad=2)),
    (4, 4, 64, 64, enchip.ROPE_HALF, 1, 21, dict(off=1)),             # 4-byte aligned
    (4, 4, 64, 64, enchip.ROPE_HALF, 1, 21, dict(off=2, pad=2)),
    (4, 4, 64, 64, enchip.ROPE_HALF, 2, 21, dict(inplace=True, pad=64)),
    (4, 4, 64, 20, enchip.ROPE_INTERLEAVED, 2, 21, dict(inplace=True, pad=5)),
    (4, 2, 64, 64, enchip.ROPE_HALF, 2, 21, dict(pos0=100000, mscale=1.25)),
    (2, 2, 32, 32, enchip.ROPE_HALF, 1, 1000, dict(eps=1e-5)),
])
def test_rows(ctx, qh, kh, hd, rot, layout, nseq, L, k):
    say(f"head_norm q={qh} k={kh} hd={hd} rot={rot} layout={layout} rows={nseq}x{L} {k}")
    check(ctx, qh, kh, hd, rot, layout, nseq, L, **k)


@pytest.mark.parametrize("layout", [enchip.ROPE_HALF, enchip.ROPE_INTERLEAVED])
def test_positions(ctx, layout):
    g = np.random.default_rng(5)
    pos = g.integers(-(2 ** 31), 2 ** 31 - 1, 77)
    pos[:4] = 0, 0, -1, 2 ** 31 - 1
    # far positions of exact frequencies: the oracle's float64 angle is exact where f is a power of two
    f = 2.0 ** -np.arange(16)
    say(f"head_norm positions layout={layout}")
    check(ctx, 3, 2, 48, 32, layout, 1, 77, pos=pos, freqs=f)


def test_sizes_of_values(ctx):
    # sums of squares past 32 bits, subnormal values, zeros, one large among small
    g = np.random.default_rng(6)
    x = g.standard_normal((8, 3 * 64)).astype(np.float32)
    x[0] *= np.float32(1e30)
    x[1] *= np.float32(3e37)
    x[2] *= np.float32(1e-20)
    x[3] *= np.float32(1e-42)
    x[4] = 0
    x[5, 7] = 1e25
    x[6, :64] = 0
    say("head_norm values of every size")
    for eps in (2.0 ** -100, 1e-6, 2.0 ** 100):
        check(ctx, 2, 1, 64, 64, enchip.ROPE_HALF, 1, 8, x=x, eps=eps)


def test_not_finite_stays_in_its_head(ctx):
    g = np.random.default_rng(7)
    x = g.standard_normal((6, 4 * 32)).astype(np.float32)
    x[1, 40] = np.inf
    x[2, 5] = np.nan
    x[3, 127] = -np.inf
    say("head_norm infinities and NaN")
    for inplace in (False, True):
        got, y, tol = run(ctx, 3, 1, 32, 0, enchip.ROPE_HALF, 1, 6, x=x, inplace=inplace)
        hit = np.zeros((6, 4), bool)
        hit[1, 1] = hit[2, 0] = hit[3, 3] = True
        fine = ~np.repeat(hit, 32, axis=1)
        assert (np.abs(got - y) <= tol)[fine].all()
        assert np.isnan(got[1, 40]) and np.isnan(got[2, :32]).all() and np.isnan(got[3, 127])
        assert (got[1, 32:64][np.arange(32) != 8] == 0).all()


def test_streams_and_graph(ctx):
    import torch

    s = torch.cuda.Stream()
    qh, kh, hd, rows = 4, 2, 64, 37
    W = (qh + kh) * hd
    gain = torch.ones(hd, device="cuda") * 1.5
    r = ctx.rope(hd)
    x, y, e = (torch.empty((rows, W), device="cuda") for _ in range(3))
    torch.cuda.synchronize()

    def call(out):
        ctx.head_norm_rope_rows_dev(r, enchip.ROPE_HALF, x.data_ptr(), W, out.data_ptr(), W, 1, rows, qh, kh, hd, gain.data_ptr(),
                                    gain.data_ptr(), 1e-6, stream=s.cuda_stream)

    try:
        with torch.cuda.stream(s):
            x.normal_()
        call(e)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            call(y)
        say("head_norm captured, 3 replays")
        for i in range(3):
            with torch.cuda.stream(s):
                x.normal_().mul_(1.0 + i)
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            call(e)
            torch.cuda.synchronize()
            assert torch.equal(y, e)
        del gr
    finally:
        ctx.release_rope(r)


def test_refusals(ctx):
    import torch

    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    r = ctx.rope(32)

    def call(rope=r, layout=enchip.ROPE_HALF, x=p, ldx=128, y=p + 8192, ldy=128, nseq=1, L=2, qh=2, kh=2, hd=32, gq=p, gk=p, eps=1e-6,
             pos0=0):
        ctx.head_norm_rope_rows_dev(rope, layout, x, ldx, y, ldy, nseq, L, qh, kh, hd, gq, gk, eps, 0, pos0)

    try:
        call()
        call(L=0), call(nseq=0), call(qh=0, kh=0), call(kh=0, gk=0), call(qh=0, gq=0), call(rope=None, layout=9, pos0=2 ** 40)
        for k in (dict(layout=2), dict(ldx=127), dict(ldy=127), dict(nseq=-1), dict(L=-1), dict(qh=-1), dict(kh=-1), dict(hd=31),
                  dict(hd=0), dict(hd=1025, ldx=8192, ldy=8192), dict(gq=0), dict(gk=0), dict(x=0), dict(y=0), dict(eps=0.0),
                  dict(eps=-1.0), dict(eps=float("nan")), dict(eps=2.0 ** 101), dict(y=p, ldy=256), dict(pos0=2 ** 40),
                  dict(qh=65536, kh=1, hd=32, ldx=2 ** 22, ldy=2 ** 22), dict(nseq=2 ** 31, L=1), dict(nseq=65536, L=65536),
                  dict(rope=None, hd=0)):
            with pytest.raises(enchip.EnchipError) as err:
                call(**k)
            assert err.value.code == enchip.ERR_ARG, k
        with pytest.raises(enchip.EnchipError) as err:
            call(rope=enchip.Rope(10 ** 9, 32))
        assert err.value.code == enchip.ERR_HANDLE
        torch.cuda.synchronize()
    finally:
        ctx.release_rope(r)
