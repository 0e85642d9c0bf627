"""Rotary, gated encoders: the new operators together, as a forward pass uses them.

DeviceBert with rope and gated layers against a float64 composition of the same W8A8 arithmetic, and
a layer of 4-bit weights (products, rotary positions, attention, gated projection) against float64."""
import math

import numpy as np
import pytest

from aikit_amd import enchip, workloads
from aikit_amd.bert_dev import LN_EPS, DeviceBert
from weight_only_oracle import act64, weight4

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


def linear64(x, lw):
    """The W8A8 linear of float64 rows: codes as the format has them, in f32 operations."""
    wq, ws, b, _ = lw
    a = x.astype(np.float32)
    m = np.abs(a).max(axis=1)
    s = (m.astype(np.float64) / 127).astype(np.float32)
    inv = np.where(s > 0, 1.0 / np.where(s > 0, s, 1).astype(np.float64), 0).astype(np.float32)
    v = (a * inv[:, None]).astype(np.float64)
    q = np.clip(np.trunc(v + np.copysign(0.5, v)), -127, 127)
    return (q @ wq.astype(np.float64).T) * s.astype(np.float64)[:, None] * ws.astype(np.float64) + b.astype(np.float64)


def ln64(x, ln):
    d = x - x.mean(axis=1, keepdims=True)
    return d / np.sqrt((d * d).mean(axis=1, keepdims=True) + LN_EPS) * ln[0].astype(np.float64) + ln[1].astype(np.float64)


def rope64(x, S, L, heads, hd, rot, layout, base=1e4):
    h = x.reshape(S, L, heads, hd).copy()
    f = base ** (-np.arange(0, rot, 2) / rot)
    a = np.arange(L)[:, None] * f
    c, s = np.cos(a)[None, :, None], np.sin(a)[None, :, None]
    i = np.arange(rot // 2)
    i, k = (i, i + rot // 2) if layout == enchip.ROPE_HALF else (2 * i, 2 * i + 1)
    x1, x2 = h[..., i].copy(), h[..., k].copy()
    h[..., i], h[..., k] = x1 * c - x2 * s, x2 * c + x1 * s
    return h.reshape(S * L, heads * hd)


def attention64(q, k, v, S, L, H, hd):
    out = np.empty_like(q)
    for z in range(S):
        r = slice(z * L, (z + 1) * L)
        for h in range(H):
            c = slice(h * hd, (h + 1) * hd)
            p = q[r, c] @ k[r, c].T / math.sqrt(hd)
            p = np.exp(p - p.max(axis=1, keepdims=True))
            out[r, c] = (p / p.sum(axis=1, keepdims=True)) @ v[r, c]
    return out


def layers_of(g, n, D, I, act):
    out = []
    for _ in range(n):
        lw = {}
        for name, K, N, a in (("qkv", D, 3 * D, enchip.ACT_NONE), ("o", D, D, enchip.ACT_NONE), ("ffn_gate", D, I, act),
                              ("ffn_up", D, I, enchip.ACT_NONE), ("ffn_down", I, D, enchip.ACT_NONE)):
            w = (g.standard_normal((N, K)) * 0.05).astype(np.float32)
            lw[name] = (*workloads.quantize_weights(w), (g.standard_normal(N) * 0.02).astype(np.float32), a)
        for name in ("attn_ln", "out_ln"):
            lw[name] = ((1 + 0.1 * g.standard_normal(D)).astype(np.float32), (0.1 * g.standard_normal(D)).astype(np.float32))
        out.append(lw)
    return out


@pytest.mark.parametrize("S,L,rot,layout,act", [(2, 16, 32, enchip.ROPE_HALF, "silu"), (4, 77, 32, enchip.ROPE_INTERLEAVED, "silu"),
                                                (3, 130, 16, enchip.ROPE_HALF, "gelu"), (1, 1, 32, enchip.ROPE_HALF, "silu")])
def test_device_forward(ctx, S, L, rot, layout, act):
    import torch

    H, hd, I = 4, 32, 384
    D = H * hd
    g = np.random.default_rng(S * L)
    layers = layers_of(g, 3, D, I, {"silu": enchip.ACT_SILU, "gelu": enchip.ACT_GELU}[act])
    rope = ctx.rope(rot)
    model = DeviceBert(ctx, layers, D, H, I, rope=rope, rope_layout=layout)
    say(f"rotary gated forward S={S} L={L} rot={rot} {act}")
    try:
        x = g.standard_normal((S * L, D)).astype(np.float32)
        s = torch.cuda.Stream()
        h = torch.from_numpy(x).cuda()
        pooled = torch.empty((S, D), device="cuda")
        torch.cuda.synchronize()
        model.embed(h, S, L, pooled, s.cuda_stream)
        torch.cuda.synchronize()
        got, gp = h.cpu().numpy(), pooled.cpu().numpy()
        y = x.astype(np.float64)
        for lw in layers:
            qkv = linear64(y, lw["qkv"])
            q, k, v = (qkv[:, i * D:(i + 1) * D] for i in range(3))
            q, k = (rope64(t, S, L, H, hd, rot, layout) for t in (q, k))
            y = ln64(y + linear64(attention64(q, k, v, S, L, H, hd), lw["o"]), lw["attn_ln"])
            inter = act64(act, linear64(y, lw["ffn_gate"])) * linear64(y, lw["ffn_up"])
            y = ln64(y + linear64(inter, lw["ffn_down"]), lw["out_ln"])
        want = y.reshape(S, L, D).mean(axis=1)
        want /= np.linalg.norm(want, axis=1, keepdims=True)
        # a code on a rounding border moves by one step of 127: the encoders' own bars
        assert np.min((gp * want).sum(axis=1)) >= 0.9999
        assert np.linalg.norm(got - y) <= 3e-2 * np.linalg.norm(y)
        # captured, and replayed between eager passes
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            model.embed(h, S, L, pooled, s.cuda_stream)
        for r in range(3):
            h.copy_(torch.from_numpy(x))
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            assert np.array_equal(pooled.cpu().numpy(), gp), r
            h.copy_(torch.from_numpy(x))
            torch.cuda.synchronize()
            model.embed(h, S, L, pooled, s.cuda_stream)
            torch.cuda.synchronize()
            assert np.array_equal(pooled.cpu().numpy(), gp), r
        del gr
    finally:
        model.close()
        ctx.release_rope(rope)


def test_gated_layer_needs_a_plain_up_projection(ctx):
    g = np.random.default_rng(1)
    lw = layers_of(g, 1, 64, 64, enchip.ACT_SILU)
    lw[0]["ffn_up"] = (*lw[0]["ffn_up"][:3], enchip.ACT_GELU)
    with pytest.raises(ValueError, match="ffn_gate"):
        DeviceBert(ctx, lw, 64, 2, 64)


@pytest.mark.parametrize("S,L", [(1, 1), (1, 7), (2, 40), (3, 200)])
def test_layer_of_4bit_weights(ctx, S, L):
    import torch

    H, hd, I, group = 4, 64, 640, 32
    D, M = H * hd, S * L
    g = np.random.default_rng(M)
    shapes = {"qkv": (3 * D, D), "o": (D, D), "gate": (I, D), "up": (I, D), "down": (D, I)}
    made = {n: weight4(g, N, K, group) for n, (N, K) in shapes.items()}
    w = {n: ctx.register_weight4(c, s, shapes[n][1], group) for n, (c, s, _) in made.items()}
    rope = ctx.rope(hd, scaling=enchip.ROPE_NONE)
    say(f"4-bit layer S={S} L={L}")
    try:
        x = g.standard_normal((M, D)).astype(np.float32)
        st = torch.cuda.Stream()
        h = torch.from_numpy(x).cuda()
        qkv, att, y, inter = (torch.empty((M, n), device="cuda") for n in (3 * D, D, D, I))
        one, zero = torch.ones(D, device="cuda"), torch.zeros(D, device="cuda")
        torch.cuda.synchronize()
        s, q = st.cuda_stream, qkv.data_ptr()
        ctx.matmul_bt_q4_dev(w["qkv"], h.data_ptr(), D, M, q, 3 * D, stream=s)
        ctx.rope_rows_dev(rope, enchip.ROPE_HALF, q, 3 * D, q, 3 * D, S, L, 2 * H, hd, stream=s)
        ctx.attention_f32_dev(q, q + 4 * D, q + 8 * D, 3 * D, att.data_ptr(), D, S, L, H, hd, 1 / math.sqrt(hd), stream=s)
        ctx.matmul_bt_q4_dev(w["o"], att.data_ptr(), D, M, y.data_ptr(), D, stream=s)
        ctx.residual_layer_norm_dev(h.data_ptr(), D, y.data_ptr(), D, M, D, one.data_ptr(), zero.data_ptr(), LN_EPS, stream=s)
        ctx.gated_q4_dev(w["gate"], w["up"], h.data_ptr(), D, M, 0, 0, enchip.ACT_SILU, inter.data_ptr(), I, stream=s)
        ctx.matmul_bt_q4_dev(w["down"], inter.data_ptr(), I, M, y.data_ptr(), D, stream=s)
        ctx.residual_layer_norm_dev(h.data_ptr(), D, y.data_ptr(), D, M, D, one.data_ptr(), zero.data_ptr(), LN_EPS, stream=s)
        torch.cuda.synchronize()
        v = {n: m[2] for n, m in made.items()}
        a = x.astype(np.float64)
        t = a @ v["qkv"].T
        qk, vv = t[:, :2 * D], t[:, 2 * D:]
        qk = rope64(qk, S, L, 2 * H, hd, hd, enchip.ROPE_HALF)
        c = attention64(qk[:, :D], qk[:, D:], vv, S, L, H, hd)
        ident = (np.ones(D), np.zeros(D))
        a = ln64(a + c @ v["o"].T, ident)
        a = ln64(a + (act64("silu", a @ v["gate"].T) * (a @ v["up"].T)) @ v["down"].T, ident)
        # the attention's gate, 2e-4 of its values, is the loosest step; LayerNorm carries it on at its own scale
        assert np.linalg.norm(h.cpu().numpy() - a) <= 4e-4 * np.linalg.norm(a)
    finally:
        for t in w.values():
            ctx.release_weight4(t)
        ctx.release_rope(rope)
