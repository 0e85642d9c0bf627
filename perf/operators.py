"""The operators of gated, rotary encoders, as cases that can be timed and compared.

One case is one pass through an operator on one GPU:

  rope    rotary positions of the query and key heads of fused [tokens, 3D] QKV rows
  q4      a[M, K] times a 4-bit weight with group scales, activations in f32
  gated   act(a Wg^T + bg) * (a Wu^T + bu), with `form`
            q8    int8 weights, activations in f32
            q4    4-bit weights with group scales, activations in f32
            w8a8  int8 weights, activations quantized per token

``run`` computes them in elementary torch operations where ``own`` is false, and through
``aikit_amd.enchip`` where it is true. A program keeps its weights registered and its rotary
frequencies made; so does this file. Calls run on the context's own stream. Inputs come from
the seed alone.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_ctx = None


def context():
    """The process's one context."""
    global _ctx
    if _ctx is None:
        from aikit_amd import enchip

        _ctx = enchip.Context(0)
    return _ctx


# ---------------------------------------------------------------------------- the cases


def listed():
    return [
        # a short query's 16 tokens at a small embedding model's width: latency
        dict(name="rope_s1l16", kind="rope", S=1, L=16, heads=12, hd=32, rot=32, layout="half", base=10000.0, scaling="none",
             factor=1.0, orig=0, packed=False),
        # bulk embedding: the benchmark's 64 x 512 tokens
        dict(name="rope_s64l512", kind="rope", S=64, L=512, heads=12, hd=64, rot=64, layout="half", base=10000.0,
             scaling="none", factor=1.0, orig=0, packed=False),
        # documents of many lengths packed behind each other, far past the trained length: part of
        # each head, neighbouring pairs, a position per row
        dict(name="rope_packed_yarn", kind="rope", S=1, L=20011, heads=16, hd=64, rot=32, layout="interleaved", base=10000.0,
             scaling="yarn", factor=16.0, orig=2048, packed=True),
        # one token through a gated FFN of int8 weights: all of it is reading the weights
        dict(name="gated_q8_m1", kind="gated", form="q8", M=1, K=1024, N=4096, act="silu", bias=False),
        # one full-length sequence through it
        dict(name="gated_q8_m512", kind="gated", form="q8", M=512, K=768, N=2304, act="silu", bias=False),
        # a short query through a small model's gated FFN, W8A8
        dict(name="gated_w8a8_m16", kind="gated", form="w8a8", M=16, K=384, N=1536, act="silu", bias=True),
        # a ragged batch and widths that are a multiple of nothing, GELU gate
        dict(name="gated_w8a8_m1500_odd", kind="gated", form="w8a8", M=1500, K=1000, N=1001, act="gelu", bias=True),
        # a full batch (64 x 512 tokens) at a large encoder's widths
        dict(name="gated_w8a8_m32768", kind="gated", form="w8a8", M=32768, K=1024, N=4096, act="silu", bias=False),
        # one token through a gated FFN of 4-bit weights
        dict(name="gated_q4_m1", kind="gated", form="q4", M=1, K=1024, N=4096, group=32, act="silu", bias=False),
        # one token through a wide 4-bit linear
        dict(name="q4_m1_wide", kind="q4", M=1, K=8192, N=8192, group=128),
        # a short query, a last group that is not whole, an odd output width
        dict(name="q4_m16_odd", kind="q4", M=16, K=1000, N=1001, group=32),
        # one full-length sequence through a 4-bit FFN-up
        dict(name="q4_m512", kind="q4", M=512, K=1024, N=4096, group=64),
    ]


COST = 32768 * 1024 * 4096 * 2  # products of the largest listed case


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer width: one a model has, or any multiple of 4, or (rarely) an odd one."""
    t = rng.random()
    if t < 0.5:
        return rng.choice([w for w in (384, 768, 1024, 1536, 2304, 4096, 8192) if lo <= w <= hi])
    w = _log(rng, lo, hi)
    return w if t > 0.85 else max(4, w // 4 * 4)


def draw(rng):
    kind = rng.choice(["rope", "gated", "gated", "q4"])
    if kind == "rope":
        hd = rng.choice([32, 64, 128])
        T, L = _log(rng, 1, 32768), _log(rng, 1, 32768)
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return dict(kind=kind, S=max(1, T // L), L=min(T, L), heads=rng.choice([12, 16]) * 64 // max(64, hd), hd=hd,
                    rot=rng.choice([hd, hd // 2, 2 * rng.randint(2, hd // 2)]), layout=rng.choice(["half", "interleaved"]),
                    base=rng.choice([1e4, 1e6]), scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 16.0]),
                    orig=2048, packed=rng.random() < 0.5)
    if kind == "q4":
        K, N = _width(rng, 256, 8192), _width(rng, 256, 8192)
        return dict(kind=kind, M=_log(rng, 1, min(4096, COST // (K * N))), K=K, N=N, group=rng.choice([32, 64, 128]))
    form, K, N = rng.choice(["q8", "q4", "w8a8"]), _width(rng, 256, 4096), _width(rng, 256, 4096)
    case = dict(kind=kind, form=form, M=_log(rng, 1, min(32768 if form == "w8a8" else 4096, COST // (2 * K * N))), K=K, N=N,
                act=rng.choice(["silu", "silu", "gelu"]), bias=rng.random() < 0.5)
    if form == "q4":
        case["group"] = rng.choice([32, 64, 128])
    return case


# ---------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)


def _randn(g, *shape, std=1.0):
    x = torch.randn(shape, device="cuda", generator=g)
    return x if std == 1.0 else x * std


def _activations(g, M, K):
    """N(0, 1) with 1% of the elements 20 times larger: an encoder's outlier channels."""
    a = _randn(g, M, K)
    return torch.where(torch.rand((M, K), device="cuda", generator=g) < 0.01, a * 20.0, a)


def _weight8(g, N, K):
    """A trained linear's int8 weight: codes of normal rows and a scale per output channel."""
    w = _randn(g, N, K, std=0.02)
    s = w.abs().amax(dim=1) / 127.0
    return torch.round(w / s[:, None]).clamp(-127, 127).to(torch.int8), s


def _weight4(g, N, K, group):
    """The same at 4 bits: two codes of c - 8 a byte, the lower k in the low half, and an f16
    scale for every `group` k's of a channel."""
    G = -(-K // group)
    w = torch.zeros((N, G * group), device="cuda")
    w[:, :K] = _randn(g, N, K, std=0.02)
    w = w.reshape(N, G, group)
    s = (w.abs().amax(dim=2) / 7.0).half()
    c = (torch.round(w / s.float()[:, :, None]).clamp(-8, 7) + 8).reshape(N, G * group)[:, :K].to(torch.uint8)
    if K % 2:
        c = torch.nn.functional.pad(c, (0, 1), value=8)
    return c[:, 0::2] | (c[:, 1::2] << 4), s


def _inputs(case, seed):
    """The case's inputs as GPU tensors, from the seed alone."""
    g = _gen(seed)
    if case["kind"] == "rope":
        T = case["S"] * case["L"]
        pos = None
        if case["packed"]:  # documents of a few hundred to a few thousand rows, each counted from its start
            starts = torch.rand(T, device="cuda", generator=g) < 1 / 2000
            starts[0] = True
            at = torch.arange(T, device="cuda")
            pos = (at - torch.cummax(torch.where(starts, at, torch.zeros_like(at)), 0).values).to(torch.int32)
            pos += torch.randint(0, 100000, (1,), device="cuda", dtype=torch.int32, generator=g)
        return dict(qkv=_randn(g, T, 3 * case["heads"] * case["hd"]), pos=pos)
    M, K, N = case["M"], case["K"], case["N"]
    x = dict(a=_activations(g, M, K))
    if case["kind"] == "q4":
        x["w"] = _weight4(g, N, K, case["group"])
        return x
    for name in ("gate", "up"):
        x[name] = _weight4(g, N, K, case["group"]) if case["form"] == "q4" else _weight8(g, N, K)
        x["b" + name] = _randn(g, N, std=0.1) if case["bias"] else None
    return x


class _Handle:
    """What a program registers once, released with the state that holds it."""

    def __init__(self, made, release):
        self.h, self._release = made, release

    def __del__(self):
        try:
            self._release(self.h)
        except Exception:
            pass


def _register(case, w):
    c = context()
    codes, scales = (t.cpu().numpy() for t in w)
    if codes.dtype == np.uint8:
        return _Handle(c.register_weight4(codes, scales, case["K"], case["group"]), c.release_weight4)
    return _Handle(c.register_weight(codes, scales), c.release_weight)


def prepare(case, seed):
    x = _inputs(case, seed)
    st = dict(case=case, x=x)
    if own:
        from aikit_amd import enchip

        c = context()
        if case["kind"] == "rope":
            scaling = dict(none=enchip.ROPE_NONE, linear=enchip.ROPE_LINEAR, ntk=enchip.ROPE_NTK, yarn=enchip.ROPE_YARN)
            st["rope"] = _Handle(c.rope(case["rot"], base=case["base"], scaling=scaling[case["scaling"]],
                                        factor=case["factor"], orig_len=case["orig"]), c.release_rope)
            st["layout"] = dict(half=enchip.ROPE_HALF, interleaved=enchip.ROPE_INTERLEAVED)[case["layout"]]
            st["out"] = torch.empty((case["S"] * case["L"], 2 * case["heads"] * case["hd"]), device="cuda")
        else:
            for name in ("w", "gate", "up"):
                if name in x:
                    st[name] = _register(case, x[name])
            st["out"] = torch.empty((case["M"], case["N"]), device="cuda")
            if case["kind"] == "gated":
                st["act"] = dict(silu=enchip.ACT_SILU, gelu=enchip.ACT_GELU)[case["act"]]
        torch.cuda.synchronize()  # the context's stream does not wait for torch's
    return st


# ---------------------------------------------------------------------------- the plain forms


def _freqs(case):
    """The rotary frequencies [rot / 2] in 64 bits, and what the rotated values are scaled by."""
    r, s, base = case["rot"], case["factor"], case["base"]
    if case["scaling"] == "ntk" and r > 2:
        base = base * s ** (r / (r - 2))
    f = torch.pow(base, -torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "yarn":
        keep = ((case["orig"] * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
        return f * keep + f / s * (1.0 - keep), 0.1 * math.log(s) + 1.0
    return f, 1.0


def _rope(case, qkv, pos):
    T, H, hd, r = case["S"] * case["L"], 2 * case["heads"], case["hd"], case["rot"]
    x = qkv[:, :H * hd].reshape(T, H, hd)
    if pos is None:
        pos = torch.arange(case["L"], device="cuda").repeat(case["S"])
    f, m = _freqs(case)
    angle = pos.double()[:, None] * f  # far positions: 64 bits
    c, s = (torch.cos(angle) * m).float()[:, None, :], (torch.sin(angle) * m).float()[:, None, :]
    if case["layout"] == "half":
        x1, x2 = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([x1 * c - x2 * s, x2 * c + x1 * s, x[..., r:]], dim=-1)
    else:
        x1, x2 = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.cat([torch.stack([x1 * c - x2 * s, x2 * c + x1 * s], dim=-1).reshape(T, H, r), x[..., r:]], dim=-1)
    return y.reshape(T, H * hd)


def _wide(case, w):
    """A registered weight's values in 32 bits: int8 codes as they are, 4-bit ones scaled (exactly)."""
    codes, scales = w
    if codes.dtype == torch.int8:
        return codes.float()
    q = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1)[:, :case["K"]].float() - 8.0
    return q * scales.float().repeat_interleave(case["group"], dim=1)[:, :case["K"]]


def _quantized(a):
    """Each row's codes and scale, as the format has them: scale = absmax / 127, codes rounded half
    away from zero."""
    m = a.abs().amax(dim=1)
    s = (m.double() / 127.0).float()  # quotients rounded once
    inv = torch.where(s == 0, torch.zeros_like(s), (1.0 / s.double()).float())
    v = (a * inv[:, None]).double()
    return torch.trunc(v + torch.copysign(torch.full_like(v, 0.5), v)).clamp(-127, 127).float(), s


def _projection(case, x, name):
    y = x["a"]
    if case["form"] == "w8a8":
        y, s = _quantized(y)
    y = y @ _wide(case, x[name]).t()
    if case["form"] == "w8a8":
        y = y * s[:, None]
    if case["form"] != "q4":
        y = y * x[name][1]
    return y if x["b" + name] is None else y + x["b" + name]


def _act(name, g):
    if name == "silu":
        return g / (1.0 + torch.exp(-g))
    return 0.5 * g * (1.0 + torch.erf(g * math.sqrt(0.5)))


def run(st):
    case, x = st["case"], st["x"]
    if not own:
        if case["kind"] == "rope":
            return _rope(case, x["qkv"], x["pos"])
        if case["kind"] == "q4":
            return x["a"] @ _wide(case, x["w"]).t()
        return _act(case["act"], _projection(case, x, "gate")) * _projection(case, x, "up")
    c, out = context(), st["out"]
    if case["kind"] == "rope":
        H, hd = case["heads"], case["hd"]
        c.rope_rows_dev(st["rope"].h, st["layout"], x["qkv"].data_ptr(), 3 * H * hd, out.data_ptr(), 2 * H * hd, case["S"],
                        case["L"], 2 * H, hd, d_pos=0 if x["pos"] is None else x["pos"].data_ptr())
        return out
    M, K, N, a = case["M"], case["K"], case["N"], x["a"].data_ptr()
    if case["kind"] == "q4":
        c.matmul_bt_q4_dev(st["w"].h, a, K, M, out.data_ptr(), N)
        return out
    bg, bu = (0 if x[b] is None else x[b].data_ptr() for b in ("bgate", "bup"))
    if case["form"] == "w8a8":
        c.w8a8_gated_dev(st["gate"].h, st["up"].h, a, M, bg, bu, st["act"], out.data_ptr())
    else:
        call = c.gated_q8_dev if case["form"] == "q8" else c.gated_q4_dev
        call(st["gate"].h, st["up"].h, a, K, M, bg, bu, st["act"], out.data_ptr(), N)
    return out


# ---------------------------------------------------------------------------- accounting


def work(case):
    if case["kind"] == "rope":
        T, H = case["S"] * case["L"], 2 * case["heads"]
        return {"bytes": 8 * T * H * case["hd"] + (4 * T if case["packed"] else 0), "flops": 3 * T * H * case["rot"]}
    M, K, N, n = case["M"], case["K"], case["N"], 1 if case["kind"] == "q4" else 2
    weight = N * -(-K // 2) + 2 * N * -(-K // case["group"]) if "group" in case else N * K + 4 * N
    return {"bytes": 4 * M * K + n * weight + (8 * N if case.get("bias") else 0) + 4 * M * N, "flops": 2 * n * M * N * K}


# ---------------------------------------------------------------------------- 64-bit results


def _rope64(case, x):
    T, H, hd, r = case["S"] * case["L"], 2 * case["heads"], case["hd"], case["rot"]
    y = x["qkv"].double()[:, :H * hd].reshape(T, H, hd).clone()
    p = (x["pos"] if x["pos"] is not None else torch.arange(T, device="cuda") % case["L"]).double()
    s, m = case["factor"], 1.0
    for j in range(r // 2):
        theta = case["base"] ** (-2.0 * j / r)
        if case["scaling"] == "linear":
            theta = theta / s
        elif case["scaling"] == "ntk" and r > 2:
            theta = (case["base"] * s ** (r / (r - 2.0))) ** (-2.0 * j / r)
        elif case["scaling"] == "yarn":
            turns = case["orig"] * theta / (2.0 * math.pi)
            ramp = 0.0 if turns < 1.0 else 1.0 if turns > 32.0 else (turns - 1.0) / 31.0
            theta, m = (1.0 - ramp) * theta / s + ramp * theta, 0.1 * math.log(s) + 1.0
        i, k = (j, j + r // 2) if case["layout"] == "half" else (2 * j, 2 * j + 1)
        z = torch.complex(y[..., i], y[..., k]) * torch.polar(torch.full_like(p, m), p * theta)[:, None]
        y[..., i], y[..., k] = z.real, z.imag
    return y.reshape(T, H * hd)


def _codes64(a):
    m = a.abs().amax(dim=1).double()
    s = (m / 127.0).float()
    r = torch.where(s > 0, 1.0 / s.double(), torch.zeros_like(m)).float()
    v = (a * r[:, None]).double()
    return torch.where(v < 0, -torch.floor(0.5 - v), torch.floor(0.5 + v)).clamp(-127, 127), s.double()


def _weight64(case, w):
    codes, scales = w
    if codes.dtype == torch.int8:
        return codes.double() * scales.double()[:, None]
    q = torch.empty((codes.shape[0], 2 * codes.shape[1]), device="cuda", dtype=torch.float64)
    q[:, 0::2], q[:, 1::2] = (codes % 16).double() - 8, (codes // 16).double() - 8
    k = torch.arange(case["K"], device="cuda") // case["group"]
    return q[:, :case["K"]] * scales.double()[:, k]


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "rope":
        return _rope64(case, x)
    if case["kind"] == "q4":
        return torch.mm(x["a"].double(), _weight64(case, x["w"]).t().contiguous())
    w = {n: _weight64(case, x[n]).t().contiguous() for n in ("gate", "up")}
    out = []
    for r in range(0, case["M"], 8192):
        a = x["a"][r:r + 8192]
        q, s = _codes64(a) if case["form"] == "w8a8" else (a.double(), None)
        g, u = (torch.mm(q, w[n]) if s is None else torch.mm(q, w[n]) * s[:, None] for n in ("gate", "up"))
        if case["bias"]:
            g, u = g + x["bgate"].double(), u + x["bup"].double()
        out.append((g * torch.sigmoid(g) if case["act"] == "silu" else g * torch.special.ndtr(g)) * u)
    return torch.cat(out)
