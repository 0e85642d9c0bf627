"""More spans, or query blocks of them, than one launch holds."""
import numpy as np
import pytest

from aikit_amd import enchip
from block_oracle import attention

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


@pytest.mark.parametrize("hd,heads,kv,nseq", [(32, 32, 32, 2 ** 22), (64, 48, 12, 2 ** 21 + 77), (128, 32, 32, 2 ** 22 - 1), (128, 64, 8, 2 ** 21 + 5)])
def test_attention_in_ranges_of_query_blocks(ctx, hd, heads, kv, nseq):
    import torch

    say(f"attention_bias {nseq} spans, most of them empty, {heads} heads of {hd} on {kv}")
    L = 1000
    sizes = {0: 5, 1: 1, 77: 30, nseq // 3: 1, nseq // 2: 70, nseq // 2 + 1: 33, nseq - 2000: 200, nseq - 1: 64}
    n = np.zeros(nseq, np.int64)
    gap = np.zeros(nseq, np.int64)
    for z, m in sizes.items():
        n[z], gap[z] = m, 7
    start = np.cumsum(gap + n) - n
    spans = np.stack([start, start + n], axis=1).astype(np.int32)
    assert spans[-1, 1] <= L
    g = np.random.default_rng(nseq)
    q, k, v = (g.standard_normal((L, h * hd)).astype(np.float32) for h in (heads, kv, kv))
    dq, dk, dv = (torch.from_numpy(x).cuda() for x in (q, k, v))
    out = torch.full((L, heads * hd), 3.0, device="cuda")
    sp = torch.from_numpy(spans).cuda()
    torch.cuda.synchronize()
    ctx.attention_bias_dev(None, dq.data_ptr(), heads * hd, dk.data_ptr(), kv * hd, dv.data_ptr(), kv * hd, out.data_ptr(), heads * hd,
                           nseq, L, heads, kv, hd, hd ** -0.5, sp.data_ptr())
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    at = [(int(spans[z, 0]), int(spans[z, 1])) for z in sorted(sizes)]
    want = attention(*(x.astype(np.float64) for x in (q, k, v)), at, heads, kv, hd, hd ** -0.5, None, np.full(got.shape, 3.0))
    inside = np.zeros(L, bool)
    for a, b in at:
        inside[a:b] = True
    assert (got[~inside] == 3.0).all()
    # as tests of single launches have it: (2 delta + (n + 64) 2^-24) max|v|, delta of sums of hd terms of at most max|q k|
    mass = hd ** -0.5 * hd * np.abs(q).max() * np.abs(k).max()
    delta = (hd * 2.0 ** -24 + 4 * 2.0 ** -22) * mass
    assert np.abs(got - want).max() <= (2 * delta + (200 + 64) * 2.0 ** -24) * np.abs(v).max()
    assert np.linalg.norm(got - want) <= 2.0 ** -17 * np.linalg.norm(want)


def test_a_number_of_sequences_past_32_bits_is_refused(ctx):
    # nothing ran, and the call said it had
    import torch

    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    for nseq in (2 ** 31, 2 ** 31 + 5, 2 ** 40):
        with pytest.raises(enchip.EnchipError) as err:
            ctx.attention_bias_dev(None, p, 32, p, 32, p, 32, p + 8192, 32, nseq, 1, 1, 1, 32, 1.0)
        assert err.value.code == enchip.ERR_ARG
    torch.cuda.synchronize()
    assert (x == 0).all()


def test_a_list_of_spans_filled_up_with_the_end(ctx):
    import torch

    say("attention_bias spans filled up with L, L")
    L, heads, hd = 300, 2, 64
    x = torch.from_numpy(np.random.default_rng(3).standard_normal((L, 3 * heads * hd)).astype(np.float32)).cuda()
    outs = []
    for spans in ([(0, 100), (100, 101), (110, 290)], [(0, 100), (100, 101), (110, 290)] + [(L, L)] * 50):
        out = torch.full((L, heads * hd), 3.0, device="cuda")
        sp = torch.tensor(spans, dtype=torch.int32, device="cuda")
        p, W = x.data_ptr(), heads * hd
        torch.cuda.synchronize()
        ctx.attention_bias_dev(None, p, 3 * W, p + 4 * W, 3 * W, p + 8 * W, 3 * W, out.data_ptr(), W, len(spans), L, heads, heads, hd, 0.125,
                               sp.data_ptr())
        torch.cuda.synchronize()
        outs.append(out.cpu().numpy())
    # the order of the sums goes by L / nseq
    assert np.linalg.norm(outs[0] - outs[1]) <= 2.0 ** -16 * np.linalg.norm(outs[0])
    assert (outs[1][101:110] == 3.0).all() and (outs[1][290:] == 3.0).all()
