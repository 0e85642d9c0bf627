"""Weights and sums of attention with a relative position bias where a bound by the largest value says little: one key far
above many others that hold all that comes out, and long rows of equal weights.

Per output, with e a key's weight relative to the row's largest, the kernel's sums S' of weights and N' of weights times
values are off from the exact S and N by
  2 delta + 2^-21 of each weight, delta the score's error: (hd 2^-24 + 3 2^-22) sum |q k| scale + 2^-22 |y| as the products
      have it and the operands' floor hd 2^-24 scale (max|q| + max|k|), doubled for 2^x,
  2^-36 a key that its two f16 parts lose below the largest, which N' alone sees, and 3 2^-22 of the second product,
  one rounding of 2^-24 for each addition."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# how the sizes choose the kernel: 8 wavefronts to 32 queries, one, tiles whole, tiles in parts, tiles in order of length
FORMS = {
    "8 wavefronts": dict(heads=1, before=299, after=0),
    "1 wavefront": dict(heads=4, before=150, after=149),
    "parts": dict(heads=2, before=0, after=0),
    "whole": dict(heads=32, before=0, after=0),
    "ordered": dict(heads=32, before=1, after=2),
}


def say(msg):
    print(f"[case] {msg}", flush=True)


def run(ctx, x, heads, hd, scale, before, after, n, kv=None, pad=0):
    """n rows among spans of no rows, every head the same columns of x [n, 3 hd]."""
    import torch

    W, kv = heads * hd, kv or heads
    one = torch.from_numpy(x).cuda()
    d = torch.cat([one[:, i * hd:(i + 1) * hd].repeat(1, k) for i, k in enumerate((heads, kv, kv))], dim=1).contiguous()
    ld, ldo = d.shape[1], W + pad
    out = torch.full((n, ldo), 3.0, device="cuda")
    spans = [(0, 0)] * before + [(0, n)] + [(n, n)] * after
    sp = torch.tensor(spans, dtype=torch.int32, device="cuda") if before + after else None
    p = d.data_ptr()
    torch.cuda.synchronize()
    ctx.attention_bias_dev(None, p, ld, p + 4 * W, ld, p + 4 * (W + kv * hd), ld, out.data_ptr(), ldo, len(spans), n, heads, kv, hd, scale,
                           0 if sp is None else sp.data_ptr())
    torch.cuda.synchronize()
    assert (out[:, W:] == 3.0).all()
    got = out[:, :W].reshape(n, heads, hd)
    assert (got == got[:, :1]).all()  # no head differs from another
    return got[:, 0].cpu().numpy()


def exact(x, hd, scale, rows):
    q, k, v = (x[:, i * hd:(i + 1) * hd].astype(np.float64) for i in range(3))
    y = scale * (q[rows] @ k.T)
    e = np.exp(y - y.max(axis=1, keepdims=True))
    mass = abs(scale) * (np.abs(q[rows]) @ np.abs(k).T)
    delta = (hd * 2.0 ** -24 + 3 * 2.0 ** -22) * mass + 2.0 ** -22 * np.abs(y) + \
        abs(scale) * hd * 2.0 ** -24 * (np.abs(q[rows]).max() + np.abs(k).max())
    return e, v, (2 * delta + 2.0 ** -21).max(axis=1, keepdims=True)


def one_above(n, hd, scale, sink, gap):
    """q, k and v of n rows: key `sink`, of value 0, has scores about `gap` above all others'."""
    g = np.random.default_rng(hd)
    x = np.zeros((n, 3 * hd), np.float32)
    x[:, 0] = 8.0
    x[:, 1:hd] = g.standard_normal((n, hd - 1)) * 0.05
    x[:, hd] = -gap / (8.0 * scale)
    x[sink, hd] = 0.0
    x[:, hd + 1:2 * hd] = g.standard_normal((n, hd - 1)) * 0.05
    x[:, 2 * hd:] = 1.0 + 0.1 * g.standard_normal((n, hd))
    x[sink, 2 * hd:] = 0.0
    return x


def held(got, x, n, hd, scale, sink, floor):
    rows = np.concatenate([np.arange(0, n, 211), [sink, n - 1]])
    e, v, rel = exact(x, hd, scale, rows)
    S, N, A = e.sum(axis=1, keepdims=True), e @ v, e @ np.abs(v)
    adds = (n / 8 + 64) * 2.0 ** -24  # of 16 keys each at least, in two parts each
    tol = ((2 * rel + 3 * 2.0 ** -22 + 2 * adds) * A + n * floor * np.abs(v).max()) / S
    assert (tol < 0.02 * N / S).all()  # far from what all of them weigh
    bad = ~(np.abs(got[rows] - N / S) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:3], got[rows][bad][:3], (N / S)[bad][:3], tol[bad][:3])


@pytest.mark.parametrize("gap", [17.0, 18.5, 20.0])
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_keys_far_below_the_largest(ctx, hd, form, gap):
    n, scale, sink = 8192 + 37, hd ** -0.5, 4000
    say(f"attention_bias one key {gap} above {n - 1} others, hd={hd}, {form}")
    x = one_above(n, hd, scale, sink, gap)
    held(run(ctx, x, hd=hd, scale=scale, n=n, **FORMS[form]), x, n, hd, scale, sink, 2.0 ** -36)


@pytest.mark.parametrize("weight", [0.7, 0.93])
@pytest.mark.parametrize("n", [8192 + 37, 2 ** 17 + 5])
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_rows_of_equal_weights(ctx, hd, form, n, weight):
    # every addition of equal numbers is rounded the same way: an error that grows with the row, if anything's does
    f, scale = FORMS[form], hd ** -0.5
    if n > 2 ** 17 and hd > 32 and f["heads"] > 4:
        f = dict(f, heads=max(12, f["heads"] * 32 // hd))
    say(f"attention_bias {n} keys of weight {weight}, hd={hd}, {form}")
    x = np.zeros((n, 3 * hd), np.float32)
    x[:, 0] = 8.0
    x[0, hd] = -np.log(weight) / (8.0 * scale)
    x[:, 2 * hd:] = 1.0
    x[:, 2 * hd + 1] = np.arange(n) % 3
    x[:, 2 * hd + 2] = np.arange(n) % 64 < 32
    x[:, 2 * hd + 3] = np.linspace(0.5, 1.5, n)
    got = run(ctx, x, hd=hd, scale=scale, n=n, **f)
    e, v, rel = exact(x, hd, scale, np.arange(1))
    want = e @ v / e.sum()
    # roundings in a sum: six for each 32 of the keys that are summed before they are set aside, three for each of those sums
    adds = (4096 / 32 * 6 + 64 + 3 * n / 4096) * 2.0 ** -24
    tol = (2 * rel + 3 * 2.0 ** -22 + 2 * adds) * want
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:3], np.abs(got / want - 1).max(), (tol / want).max())


@pytest.mark.parametrize("gap", [16.0, 17.0])
@pytest.mark.parametrize("heads", [1, 24])  # workgroups of 8 and of 16 wavefronts
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("sign", [1, -1])
def test_the_fused_attention_without_a_bias(ctx, hd, heads, gap, sign):
    import torch

    n, scale, sink = 8192 + 37, hd ** -0.5, 4000
    say(f"attention_f32 one key {gap} above {n - 1} others, hd={hd}, {heads} heads, scale {sign * scale}")
    x = one_above(n, hd, scale, sink, gap)
    one = torch.from_numpy(x).cuda()
    one[:, :hd] *= sign
    W = heads * hd
    d = torch.cat([one[:, i * hd:(i + 1) * hd].repeat(1, heads) for i in range(3)], dim=1).contiguous()
    out = torch.full((n, W), 3.0, device="cuda")
    p = d.data_ptr()
    torch.cuda.synchronize()
    ctx.attention_f32_dev(p, p + 4 * W, p + 8 * W, 3 * W, out.data_ptr(), W, 1, n, heads, hd, sign * scale)
    torch.cuda.synchronize()
    got = out.reshape(n, heads, hd)
    assert (got == got[:, :1]).all()
    held(got[:, 0].cpu().numpy(), x, n, hd, scale, sink, 2.0 ** -32)


@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_rows_into_outputs_of_any_pitch(ctx, hd, form):
    # what is set aside stands in the outputs' place
    n, scale, sink = 8192 + 37, hd ** -0.5, 4000
    say(f"attention_bias {n} rows, outputs 3 floats apart, hd={hd}, {form}")
    x = one_above(n, hd, scale, sink, 17.0)
    want = run(ctx, x, hd=hd, scale=scale, n=n, **FORMS[form])
    assert (run(ctx, x, hd=hd, scale=scale, n=n, pad=3, **FORMS[form]) == want).all()


@pytest.mark.parametrize("form", ["whole", "ordered"])
@pytest.mark.parametrize("hd,heads,kv", [(32, 64, 8), (64, 64, 16), (128, 48, 12), (64, 48, 24)])
def test_long_rows_of_heads_that_share_keys(ctx, hd, heads, kv, form):
    n, scale, sink = 8192 + 37, hd ** -0.5, 4000
    say(f"attention_bias {n} rows, {heads} heads of {hd} on {kv}, {form}")
    x = one_above(n, hd, scale, sink, 17.0)
    held(run(ctx, x, hd=hd, scale=scale, n=n, kv=kv, **dict(FORMS[form], heads=heads)), x, n, hd, scale, sink, 2.0 ** -36)
