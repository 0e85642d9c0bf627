"""Head norms, relative position bias, spans and adapters together, as a forward pass uses them: DeviceBert
against a float64 composition of the same W8A8 arithmetic, and adapters beside 4-bit and int8 weight-only products."""
import math

import numpy as np
import pytest

from aikit_amd import enchip, workloads
from aikit_amd.bert_dev import LN_EPS, DeviceBert
from block_oracle import adapters as adapters64
from block_oracle import attention, bucket_of, gelu64, head_norm_rope, linear64
from weight_only_oracle import weight4

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[case] {msg}", flush=True)


def ln64(x, ln):
    d = x - x.mean(axis=1, keepdims=True)
    return d / np.sqrt((d * d).mean(axis=1, keepdims=True) + LN_EPS) * ln[0].astype(np.float64) + ln[1].astype(np.float64)


def layers_of(g, n, D, W, I, hd, gated, norms):
    out = []
    for _ in range(n):
        lw = {}
        act = enchip.ACT_NONE if gated else enchip.ACT_GELU
        shapes = [("qkv", D, W, enchip.ACT_NONE), ("o", D, D, enchip.ACT_NONE), ("ffn_up", D, I, act), ("ffn_down", I, D, enchip.ACT_NONE)]
        if gated:
            shapes.append(("ffn_gate", D, I, enchip.ACT_SILU))
        for name, K, N, a in shapes:
            w = (g.standard_normal((N, K)) * 0.05).astype(np.float32)
            lw[name] = (*workloads.quantize_weights(w), (g.standard_normal(N) * 0.02).astype(np.float32), a)
        for name in ("attn_ln", "out_ln"):
            lw[name] = ((1 + 0.1 * g.standard_normal(D)).astype(np.float32), (0.1 * g.standard_normal(D)).astype(np.float32))
        if norms:
            for name in ("q_norm", "k_norm"):
                lw[name] = (1 + 0.2 * g.standard_normal(hd)).astype(np.float32)
        out.append(lw)
    return out


@pytest.mark.parametrize("H,KV,hd,I,gated,norms,rot,bias,low,rows,spans", [
    (4, 4, 32, 384, False, True, 32, True, ("qkv", "o", "ffn_up", "ffn_down"), (3, 40), None),
    (4, 2, 64, 512, True, True, 64, False, ("qkv", "ffn_down"), (1, 300), [(0, 7), (7, 8), (8, 8), (20, 180), (180, 300)]),
    (2, 1, 128, 320, False, True, 0, True, ("o",), (2, 50), None),
    (6, 6, 32, 384, False, False, 0, True, (), (1, 200), [(0, 33), (40, 41), (60, 200)]),
    (4, 4, 64, 1000, False, False, 32, False, ("ffn_up", "ffn_down"), (1, 90), None),
    (4, 4, 64, 384, True, False, 0, False, ("o", "qkv"), (1, 1), None),
])
def test_device_forward(ctx, H, KV, hd, I, gated, norms, rot, bias, low, rows, spans):
    import torch

    S, L = rows
    M, D, n = S * L, H * hd, 2
    W = D + 2 * KV * hd
    g = np.random.default_rng(M + H)
    layers = layers_of(g, n, D, W, I, hd, gated, norms)
    rope = ctx.rope(rot) if rot else None
    table = g.standard_normal((32, H)).astype(np.float32)
    rp = ctx.relpos(table, 50) if bias else None
    slots, r = 3, 8
    sets, made = [], []
    for lw in layers:
        a, m = {}, {}
        for name in low:
            N, K = lw[name][0].shape
            A, B = (g.standard_normal((slots, r, K)) / math.sqrt(K)).astype(np.float32), (g.standard_normal((slots, N, r)) * 0.05).astype(np.float32)
            a[name] = ctx.adapters(K, N, r, slots)
            for s in range(slots):
                ctx.set_adapter(a[name], s, A[s], B[s], 0.7)
            m[name] = (A, B)
        sets.append(a), made.append(m)
    model = DeviceBert(ctx, layers, D, H, I, rope=rope, kv_heads=KV, relpos=rp, adapters=sets if low else None)
    say(f"attention block forward H={H} KV={KV} hd={hd} gated={gated} norms={norms} rot={rot} bias={bias} {low} {rows} {spans}")
    try:
        x = g.standard_normal((M, D)).astype(np.float32)
        ids = np.repeat(g.integers(-1, slots, -(-M // 13)), 13)[:M].astype(np.int32)
        at = [(z * L, (z + 1) * L) for z in range(S)] if spans is None else spans
        pos = np.zeros(M, np.int32)
        for a, b in at:
            pos[a:b] = np.arange(b - a)
        st = torch.cuda.Stream()
        h, pooled = torch.from_numpy(x).cuda(), torch.zeros((len(at), D), device="cuda")
        k = {}
        if spans is not None:
            k = dict(spans=torch.tensor(spans, dtype=torch.int32, device="cuda"), pos=torch.from_numpy(pos).cuda())
        if low:
            k["ids"] = torch.from_numpy(ids).cuda()
        torch.cuda.synchronize()
        model.embed(h, S, L, pooled, st.cuda_stream, **k)
        torch.cuda.synchronize()
        got, gp = h.cpu().numpy(), pooled.cpu().numpy()

        def lin(li, name, y):
            lw = layers[li][name]
            out = linear64(y, *lw[:3])
            if name in made[li]:
                out = out + adapters64(y.astype(np.float32), ids, *made[li][name], [0.7] * slots)[0]
            return out

        fn = (lambda d, i: table[bucket_of(d, 32, 50), i].astype(np.float64)) if bias else None
        y = x.astype(np.float64)
        for li, lw in enumerate(layers):
            qkv = lin(li, "qkv", y)
            qk, v = qkv[:, :D + KV * hd], qkv[:, D + KV * hd:]
            if norms:
                qk, _ = head_norm_rope(qk, H, KV, hd, lw["q_norm"], lw["k_norm"], 1e-6, pos, rot, False)
            elif rot:
                f = np.cos(pos[:, None] * 1e4 ** (-np.arange(0, rot, 2) / rot)), np.sin(pos[:, None] * 1e4 ** (-np.arange(0, rot, 2) / rot))
                t = qk.reshape(M, H + KV, hd).copy()
                x1, x2 = t[..., :rot // 2].copy(), t[..., rot // 2:rot].copy()
                t[..., :rot // 2], t[..., rot // 2:rot] = x1 * f[0][:, None] - x2 * f[1][:, None], x2 * f[0][:, None] + x1 * f[1][:, None]
                qk = t.reshape(M, -1)
            c = attention(qk[:, :D], qk[:, D:], v, at, H, KV, hd, 1 / math.sqrt(hd), fn)
            y = ln64(y + lin(li, "o", c), lw["attn_ln"])
            up = lin(li, "ffn_up", y)
            inter = up * (lambda t: t / (1 + np.exp(-t)))(lin(li, "ffn_gate", y)) if gated else gelu64(up)
            y = ln64(y + lin(li, "ffn_down", inter), lw["out_ln"])
        inside = np.zeros(M, bool)
        for i, (a, b) in enumerate(at):
            inside[a:b] = True
            if b > a:
                want = y[a:b].mean(axis=0)
                # a code on a rounding border moves by one step of 127: the encoders' own bars
                assert (gp[i] * want).sum() / np.linalg.norm(want) >= 0.9999, i
            else:
                assert (gp[i] == 0).all()
        assert np.linalg.norm((got - y)[inside]) <= 3e-2 * np.linalg.norm(y[inside])
        # captured, and replayed between eager passes
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=st):
            model.embed(h, S, L, pooled, st.cuda_stream, **k)
        for rep in range(3):
            h.copy_(torch.from_numpy(x))
            torch.cuda.synchronize()
            gr.replay()
            torch.cuda.synchronize()
            assert np.array_equal(pooled.cpu().numpy(), gp), rep
        del gr
        if low:  # without ids: the model alone
            h.copy_(torch.from_numpy(x))
            k.pop("ids")
            torch.cuda.synchronize()
            model.embed(h, S, L, pooled, st.cuda_stream, **k)
            torch.cuda.synchronize()
            assert not np.array_equal(pooled.cpu().numpy(), gp) or (ids < 0).all()
    finally:
        model.close()
        for a in sets:
            for t in a.values():
                ctx.release_adapters(t)
        if rope:
            ctx.release_rope(rope)
        if rp:
            ctx.release_relpos(rp)


def test_constructor_refusals(ctx):
    g = np.random.default_rng(1)
    lw = layers_of(g, 1, 64, 192, 64, 32, True, True)
    ok = ctx.adapters(64, 64, 4, 1)
    try:
        for k, match in ((dict(kv_heads=3), "kv_heads"), (dict(adapters=[]), "layers of adapters"), (dict(adapters=[{"ffn_gate": ok}]), "ffn_gate"),
                         (dict(adapters=[{"ffn_up": ok}]), "ffn_up"), (dict(adapters=[{"qkv": ok}]), "adapters of")):
            with pytest.raises(ValueError, match=match):
                DeviceBert(ctx, lw, 64, 2, 64, **k)
        one = [dict(lw[0])]
        del one[0]["k_norm"]
        with pytest.raises(ValueError, match="q_norm"):
            DeviceBert(ctx, one, 64, 2, 64)
        bad = [dict(lw[0], q_norm=np.ones(16, np.float32))]
        with pytest.raises(ValueError, match="q_norm"):
            DeviceBert(ctx, bad, 64, 2, 64)
        import torch

        m = DeviceBert(ctx, lw, 64, 2, 64)
        h = torch.zeros((4, 64), device="cuda")
        with pytest.raises(ValueError, match="ids"):
            m.forward(h, 1, 4, ids=torch.zeros(4, dtype=torch.int32, device="cuda"))
        with pytest.raises(ValueError, match="spans"):
            m.forward(h, 1, 4, spans=torch.zeros((1, 2), device="cuda"))
        with pytest.raises(ValueError, match="pos"):
            m.forward(h, 1, 4, pos=torch.zeros(3, dtype=torch.int32, device="cuda"))
        m.close()
    finally:
        ctx.release_adapters(ok)


@pytest.mark.parametrize("M", [1, 33, 300])
def test_adapters_beside_weight_only_products(ctx, M):
    import torch

    K, N, r, slots, group = 320, 200, 12, 3, 32
    g = np.random.default_rng(M)
    say(f"adapters beside 4-bit and int8 weight-only products M={M}")
    c4, s4, v4 = weight4(g, N, K, group)
    w4 = ctx.register_weight4(c4, s4, K, group)
    wq, ws = workloads.quantize_weights((g.standard_normal((N, K)) * 0.05).astype(np.float32))
    w8 = ctx.register_weight(wq, ws)
    A, B = (g.standard_normal((slots, r, K)) / math.sqrt(K)).astype(np.float32), (g.standard_normal((slots, N, r)) * 0.1).astype(np.float32)
    h = ctx.adapters(K, N, r, slots)
    try:
        for s in range(slots):
            ctx.set_adapter(h, s, A[s], B[s], 1.5)
        a, ids = g.standard_normal((M, K)).astype(np.float32), g.integers(-1, slots, M).astype(np.int32)
        da, di, y = torch.from_numpy(a).cuda(), torch.from_numpy(ids).cuda(), torch.empty((M, N), device="cuda")
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        part, mass = adapters64(a, ids, A, B, [1.5] * slots)
        for w, v, call in ((w4, v4.astype(np.float64), ctx.matmul_bt_q4_dev), (w8, wq.astype(np.float64) * ws.astype(np.float64)[:, None], ctx.matmul_bt_q8_dev)):
            call(w, da.data_ptr(), K, M, y.data_ptr(), N, stream=st.cuda_stream)
            ctx.adapters_add_dev(h, da.data_ptr(), K, M, di.data_ptr(), y.data_ptr(), N, y.data_ptr(), N, stream=st.cuda_stream)
            torch.cuda.synchronize()
            base = a.astype(np.float64) @ v.T
            # (n + 8) 2^-24 + 2^-23 of the products' magnitudes (the products' own bound), (K + r + 4) 2^-24 of the adapters'
            tol = ((K + 8) * 2.0 ** -24 + 2.0 ** -23) * (np.abs(a).astype(np.float64) @ np.abs(v).T) + (K + r + 4) * 2.0 ** -24 * mass + \
                2.0 ** -23 * np.abs(base + part)
            assert (np.abs(y.cpu().numpy() - (base + part)) <= tol).all()
    finally:
        ctx.release_weight4(w4)
        ctx.release_weight(w8)
        ctx.release_adapters(h)
