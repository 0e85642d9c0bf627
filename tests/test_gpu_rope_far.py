"""Rotary positions far from 0: the angle p f_j of a frequency in 64 bits, reduced exactly here in whole numbers.

The tolerance holds no term in p or f. The reduced angle is rounded to f32: half a step of a value up to half
a turn, 2^-26 turns = 2^-23.3 radians; sine and cosine are within 2 ulp (2^-23), times mscale (half an ulp); two
products and their sum round once each (2^-24): under 2^-21 m (|x1| + |x2|) together."""
import numpy as np
import pytest

from aikit_amd import enchip

pytestmark = pytest.mark.gpu

BITS = 300


def pi_scaled():
    """floor(pi 2^BITS) to a few units, by Machin's formula."""
    def atan_inv(n):
        t = x = (1 << (BITS + 20)) // n
        k, sign = 3, -1
        while x:
            x //= n * n
            t += sign * (x // k)
            k, sign = k + 2, -sign
        return t

    return (4 * (4 * atan_inv(5) - atan_inv(239))) >> 20


TWO_PI = 2 * pi_scaled()


def angles(pos, freqs):
    """p f mod 2 pi, [positions, frequencies], in 64 bits."""
    out = np.empty((len(pos), len(freqs)))
    for j, f in enumerate(freqs):
        num, den = float(f).as_integer_ratio()
        for i, p in enumerate(pos):
            r = ((int(p) * num << BITS) // den) % TWO_PI
            out[i, j] = (r >> (BITS - 120)) / 2.0 ** 120
    return out


@pytest.mark.parametrize("layout", [enchip.ROPE_HALF, enchip.ROPE_INTERLEAVED])
@pytest.mark.parametrize("freqs", [[1.0, 0.37, 0.75, 1e-2, 3e-5, 0.0], [17.0, -5.5, 6.283185307179586, 1000.25, 123456.789, 1e9],
                                   [2.0 ** 40, -2.0 ** 40, 1e12, 3.3e11, 0.1, -0.7]])
def test_far_positions(ctx, layout, freqs):
    import torch

    n, hd, heads = len(freqs), 2 * len(freqs), 3
    g = np.random.default_rng(n)
    pos = np.concatenate([[0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 2, 1 << 20, 131071], g.integers(-2 ** 31, 2 ** 31, size=200)])
    x = g.standard_normal((len(pos), heads * hd)).astype(np.float32)
    r = ctx.rope_from_freqs(freqs, mscale=1.25)
    try:
        print(f"[case] rope far layout={layout} freqs={freqs}", flush=True)
        dx, dp = torch.from_numpy(x).cuda(), torch.from_numpy(pos.astype(np.int32)).cuda()
        dy = torch.empty_like(dx)
        torch.cuda.synchronize()
        ctx.rope_rows_dev(r, layout, dx.data_ptr(), heads * hd, dy.data_ptr(), heads * hd, 1, len(pos), heads, hd, dp.data_ptr())
        torch.cuda.synchronize()
        got = dy.cpu().numpy().reshape(-1, heads, hd)
    finally:
        ctx.release_rope(r)
    i = np.arange(n) if layout == enchip.ROPE_HALF else 2 * np.arange(n)
    k = i + (n if layout == enchip.ROPE_HALF else 1)
    h = x.astype(np.float64).reshape(-1, heads, hd)
    ang = angles(pos, freqs)[:, None, :]
    c, s = 1.25 * np.cos(ang), 1.25 * np.sin(ang)
    tol = 1.25 * 2.0 ** -21 * (np.abs(h[..., i]) + np.abs(h[..., k]))
    for at, want in ((i, h[..., i] * c - h[..., k] * s), (k, h[..., k] * c + h[..., i] * s)):
        err = np.abs(got[..., at] - want)
        assert np.all(err <= tol), f"worst {np.max(err / tol, axis=(0, 1))} of the bound per frequency"


def test_counted_positions_far_out(ctx):
    # positions that count up from pos0 past 32 bits
    import torch

    r = ctx.rope_from_freqs([1.0, 0.3])
    try:
        for pos0 in (2 ** 31, 2 ** 31 - 7, -2 ** 31):
            pos = pos0 + np.arange(40)
            d = torch.zeros((40, 4), device="cuda")
            d[:, :2] = 1.0
            torch.cuda.synchronize()
            ctx.rope_rows_dev(r, enchip.ROPE_HALF, d.data_ptr(), 4, d.data_ptr(), 4, 1, 40, 1, 4, pos0=pos0)
            torch.cuda.synchronize()
            got, ang = d.cpu().numpy().astype(np.float64), angles(pos, [1.0, 0.3])
            assert np.abs(got - np.concatenate([np.cos(ang), np.sin(ang)], axis=1)).max() <= 2.0 ** -21
    finally:
        ctx.release_rope(r)


def test_frequencies_past_the_range_are_refused(ctx):
    for f in (np.nextafter(2.0 ** 40, np.inf), -1e13, 1e300, -1e308):
        with pytest.raises(enchip.EnchipError) as e:
            ctx.rope_from_freqs([0.5, f])
        assert e.value.code == enchip.ERR_ARG, f
    with pytest.raises(enchip.EnchipError) as e:
        ctx.rope(64, base=1e-200)  # frequencies up to 1e194
    assert e.value.code == enchip.ERR_ARG

def test_stretched_bases_past_64_bits_are_refused(ctx):
    # base factor^(r / (r - 2)) is infinite: every frequency but the first would be 0
    with pytest.raises(enchip.EnchipError) as e:
        ctx.rope(64, base=1e300, scaling=enchip.ROPE_NTK, factor=1e30)
    assert e.value.code == enchip.ERR_ARG
    with pytest.raises(enchip.EnchipError) as e:
        ctx.rope(4, base=1e4, scaling=enchip.ROPE_NTK, factor=1e200)
    assert e.value.code == enchip.ERR_ARG
    ctx.release_rope(ctx.rope(64, base=1e300, scaling=enchip.ROPE_NTK, factor=1e6))
