"""A BERT encoder forward resident on the device, composed from libenchip's entry points.

It follows encoder/bert.go:324-368 layer for layer, with every activation kept in device
memory between operations (the residency the reference names as the next step after the
matmul seam, docs/task-native-gpu.md:418-427):

  qkv   = W8A8(h, Wqkv) + b            enchip_w8a8_linear_dev (Q, K, V fused: one N = 3D
                                        weight sharing one activation quantization,
                                        linalg.MatmulBTW8A8Batch)
  ctx_h = softmax(Q_h.K_h^T/sqrt(hd)).V_h
                                        enchip_attention_f32_dev: every (head, sequence) in
                                        one launch, heads read in place from qkv, scores
                                        kept on chip (head_dim 32/64; any L with the default
                                        online-softmax mode, L <= 512 otherwise); otherwise
                                        enchip_matmul_bt_f32_dev, enchip_softmax_rows_scaled_dev,
                                        enchip_matmul_bt_f32_dev through an [S, H, L, L] buffer
  out   = W8A8(ctx, Wo) + b             enchip_w8a8_linear_dev
  h     = LN(h + out)                   enchip_residual_layer_norm_dev
  inter = GELU(W8A8(h, Wi) + b)         enchip_w8a8_linear_dev (fused epilogue), or, when
                                        FFN-down takes fragment-major codes of K <= 4096,
                                        W8A8(h, Wi) + b alone, the GELU applied by FFN-down's
                                        quantization (enchip_quant_rows_frag_gelu_dev): the
                                        same codes
  ffn   = W8A8(inter, Wd) + b           enchip_w8a8_linear_dev
  h     = LN(h + ffn)                   enchip_residual_layer_norm_dev

A linear that takes fragment-major codes (enchip_frag_route) runs as
enchip_quant_rows_frag_dev + enchip_w8a8_pre_frag_dev into this object's code buffer: the
kernels enchip_w8a8_linear_dev launches, as two calls that can be timed apart. When the
linear after a LayerNorm (FFN-up, and the next layer's QKV) takes fragment-major
codes, the LayerNorm and that linear's quantization run as one kernel
(enchip_residual_layer_norm_quant_dev, then enchip_w8a8_pre_frag_dev): the same bits, and
the normalised rows are not read back to be quantized.

and pools with enchip_pool_mean_l2_dev (encoder/pooling.go:84-105, embed/pool.go:22-38),
or, as a cross-encoder, scores each sequence with classifier(tanh(pooler(CLS)))
(encoder/crossencoder.go:219-238): the f32 MatmulBT on the CLS rows read in place, then
enchip_bias_act_rows_dev for the bias + TanhF32 and the classifier's bias.
forward() takes the [S*L, D] f32 hidden state after the embedding LayerNorm; embeddings()
computes that state on the device from token ids (bert.go:299-323: enchip_embed_rows_dev,
then enchip_residual_layer_norm_dev with no residual). Every sequence of a batch has the
same L.

A rotary encoder passes `rope` (the query and key heads turned in place in qkv before the attention,
enchip_rope_rows_dev), a gated one layers with an "ffn_gate" beside "ffn_up": inter = act(W8A8(h, Wg)
+ bg) * (W8A8(h, Wi) + b) in enchip_w8a8_gated_dev (encoder/forward_q8.go:264-279 swigluMLPQ8 on
the NomicBERT forward's order, with W8A8 linears as in the rest of this module).

Layers with "q_norm" and "k_norm" have their query and key heads RMS-normed in qkv, turned in the same pass when
`rope` is given (enchip_head_norm_rope_rows_dev). `relpos` (a learned bias by relative position), `kv_heads` fewer
than `heads`, or sequences given as spans of rows take enchip_attention_bias_dev (heads of 32, 64 or 128; its products are
ATT_FLASH_F16's, whatever Context.set_attention_products says); embed() then
pools the spans (enchip_pool_mean_l2_spans_dev). Low-rank adapters of many requests stand beside any linear
but a gated layer's gate and up projection (`adapters`; enchip_w8a8_linear_adapters_dev): each row's by its id.

This module holds no arithmetic of its own; torch provides device buffers and the stream.
"""
from __future__ import annotations

import math
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from . import enchip

LN_EPS = 1e-12  # BERT's layer_norm_eps (encoder/bert.go)
LINEARS = ("qkv", "o", "ffn_gate", "ffn_up", "ffn_down")


class DeviceBert:
    """Weights registered once; forward() runs the layers on device tensors.

    layers: per layer {"qkv"|"o"|"ffn_up"|"ffn_down": (wq int8 [N,K], ws f32 [N],
    bias f32 [N], act), "attn_ln"|"out_ln": (gain f32 [D], shift f32 [D])}; a gated layer
    also has "ffn_gate", whose act (ACT_SILU or ACT_GELU) is the gate's, and its "ffn_up" has
    ACT_NONE. rope: rotary frequencies (Context.rope) of the context, which outlive this object,
    with rope_layout; such a model's position table (set_embeddings) is zeros.
    A layer may have "q_norm" and "k_norm" (f32 [head_dim], both or neither): gains of RMS norms of
    its query and key heads, with norm_eps. kv_heads: heads of keys and values, a divisor of heads; "qkv"
    then has hidden + 2 kv_heads head_dim rows. relpos: a bias (Context.relpos) for the attention of every
    layer. adapters: per layer a dict of Context.adapters sets by linear ("qkv", "o", "ffn_up", "ffn_down";
    not "ffn_up" of a gated layer), used where forward() is given ids. All of these outlive this object.
    """

    def __init__(self, ctx: enchip.Context, layers: Sequence[Dict], hidden: int, heads: int, ffn: int,
                 fused: bool = True, fuse_ln_quant: bool = True, gelu_in_quant: bool = True,
                 rope: Optional["enchip.Rope"] = None, rope_layout: int = enchip.ROPE_HALF,
                 kv_heads: Optional[int] = None, norm_eps: float = 1e-6, relpos: Optional["enchip.RelPos"] = None,
                 adapters: Optional[Sequence[Dict[str, "enchip.Adapters"]]] = None):
        import torch

        for lw in layers:
            if "ffn_gate" in lw and lw["ffn_up"][3] != enchip.ACT_NONE:
                raise ValueError("a gated layer's activation is its ffn_gate's: ffn_up must have ACT_NONE")

            if ("q_norm" in lw) != ("k_norm" in lw):
                raise ValueError("a layer has both q_norm and k_norm, or neither")
        if adapters is not None and len(adapters) != len(layers):
            raise ValueError(f"{len(adapters)} layers of adapters for {len(layers)} layers")
        for lw, sets in zip(layers, adapters or ()):
            for name, a in sets.items():
                if name not in ("qkv", "o", "ffn_up", "ffn_down") or (name == "ffn_up" and "ffn_gate" in lw):
                    raise ValueError(f"no adapters beside {name} here")
                if (a.N, a.K) != lw[name][0].shape:
                    raise ValueError(f"adapters of [{a.N}, {a.K}] beside {name} {lw[name][0].shape}")

        self.fused = fused
        self.fuse_ln_quant = fuse_ln_quant
        self.gelu_in_quant = gelu_in_quant
        self.rope, self.rope_layout = rope, rope_layout
        self.torch = torch
        self.ctx, self.D, self.H, self.I = ctx, hidden, heads, ffn
        self.hd = hidden // heads
        if self.hd * heads != hidden:
            raise ValueError(f"hidden {hidden} is not a multiple of heads {heads}")
        self.KV = heads if kv_heads is None else kv_heads
        if self.KV < 1 or heads % self.KV:
            raise ValueError(f"kv_heads {kv_heads} does not divide heads {heads}")
        self.W = hidden + 2 * self.KV * self.hd  # a row of qkv
        self.norm_eps, self.relpos = norm_eps, relpos
        self.adapters = [dict(a) for a in adapters] if adapters is not None else None
        self.handles: List[Dict[str, Tuple]] = []
        dev = torch.device("cuda")
        for lw in layers:
            entry = {}
            for name in LINEARS:
                if name not in lw and name == "ffn_gate":
                    continue
                wq, ws, b, act = lw[name]
                entry[name] = (ctx.register_weight(wq, ws), torch.from_numpy(np.ascontiguousarray(b)).to(dev), act)
            for name in ("q_norm", "k_norm"):
                if name in lw:
                    if np.shape(lw[name]) != (self.hd,):
                        raise ValueError(f"{name} shape {np.shape(lw[name])} is not ({self.hd},)")
                    entry[name] = torch.from_numpy(np.ascontiguousarray(lw[name], np.float32)).to(dev)
            for name in ("attn_ln", "out_ln"):
                g, s = lw[name]
                entry[name] = (torch.from_numpy(np.ascontiguousarray(g)).to(dev),
                               torch.from_numpy(np.ascontiguousarray(s)).to(dev))
            self.handles.append(entry)
        self._bufs = {}
        self._captured = []  # buffers that a graph holds the addresses of
        self._emb = None
        # Optional callback mark(label) called before each device operation this object
        # enqueues (and with "end" after the last), for per-operation timing; None: off.
        self.mark = None

    def _m(self, label: str) -> None:
        if self.mark is not None:
            self.mark(label)

    def set_embeddings(self, word, pos, ln, typ=None, pos_off: int = 0) -> None:
        """The embedding tables: word [vocab, D], pos [npos, D], optional token types
        [type_vocab, D], the embedding LayerNorm (gain [D], shift [D]), as numpy arrays
        (uploaded) or f32 device tensors; pos_off is the position-id offset (0 for BERT,
        pad_token_id + 1 for RoBERTa / XLM-R)."""
        t, dev = self.torch, self.torch.device("cuda")

        def up(a):  # numpy arrays are uploaded; f32 device tensors are used as they are
            if isinstance(a, t.Tensor):
                if a.device.type != "cuda" or a.dtype != t.float32 or not a.is_contiguous():
                    raise ValueError("set_embeddings: tensors must be contiguous f32 on the device")
                return a
            return t.from_numpy(np.ascontiguousarray(a, np.float32)).to(dev)

        self._emb = dict(word=up(word), pos=up(pos), type=None if typ is None else up(typ),
                         ln=(up(ln[0]), up(ln[1])), pos_off=int(pos_off))

    def embeddings(self, ids, S: int, L: int, h, segs=None, stream: int = 0) -> None:
        """h [S*L, D] = LayerNorm(word[id] + pos[i + pos_off] (+ type[seg])) for int32 device ids
        [S*L] (and optional int32 segment ids), bert.go:299-323."""
        e, D = self._emb, self.D
        if e is None:
            raise ValueError("embeddings: call set_embeddings first")
        typ = e["type"]
        self._m("embed_rows")
        self.ctx.embed_rows_dev(ids.data_ptr(), 0 if segs is None else segs.data_ptr(), S, L, e["word"].data_ptr(),
                                e["word"].shape[0], e["pos"].data_ptr(), e["pos"].shape[0], e["pos_off"],
                                0 if typ is None else typ.data_ptr(), 0 if typ is None else typ.shape[0], D,
                                h.data_ptr(), D, stream)
        g, b = e["ln"]
        self._m("embed_ln")
        self.ctx.residual_layer_norm_dev(h.data_ptr(), D, 0, D, S * L, D, g.data_ptr(), b.data_ptr(), LN_EPS, stream)

    def close(self) -> None:
        for entry in self.handles:
            for name in LINEARS:
                if name in entry:
                    self.ctx.release_weight(entry[name][0])
        self.handles = []
        self._bufs, self._captured = {}, []

    def bias_attention(self, spans=None) -> bool:
        """Whether the attention is enchip_attention_bias_dev's."""
        return self.relpos is not None or self.KV != self.H or spans is not None

    def fused_attention(self, L: int) -> bool:
        if self.bias_attention():
            return True
        if not self.fused or self.hd not in (32, 64):
            return False
        return L <= 512 or self.ctx.attention_products in (enchip.ATT_FLASH_BF16, enchip.ATT_FLASH_F16)

    # Widest FFN-down input whose GELU moves into the quantization: every width the
    # quantizer takes (enchip_quant_rows_frag_gelu_dev: ldq <= 4096). Measured on MI355X,
    # same process, identical outputs: BERT-base (K = 3072) 8.81 -> 8.52 ms per encode,
    # XLM-R-large (K = 4096) 53.5 -> 51.8 ms per rerank batch.
    GELU_QUANT_MAX_K = 4096

    def gelu_quant_route(self, up_act: int, down: "enchip.Weight", M: int) -> int:
        """The padded K of FFN-down's codes when FFN-up's GELU moves into FFN-down's
        quantization (enchip_quant_rows_frag_gelu_dev: FFN-up stores its pre-activations, the
        quantizer applies the GELU; the same codes, scales and outputs), else 0."""
        if not self.gelu_in_quant or up_act != enchip.ACT_GELU or down.K % 4 != 0:
            return 0
        ok, ldq = self.ctx.frag_route(down, M)
        return ldq if ok and ldq <= self.GELU_QUANT_MAX_K else 0

    def _on(self, stream: int):
        """What is allocated within belongs to `stream`, on which the layers run: torch's allocator gives it to
        another tensor only there, behind the work that is queued on it (not to the caller's tensors, whose work on
        torch's own stream nothing orders after this object's)."""
        return self.torch.cuda.stream(self.torch.cuda.ExternalStream(stream or self.ctx.stream()))

    def _buffers(self, S: int, L: int, stream: int, scores: bool = True):
        """The activations of S * L rows. Nothing is filled: rows are independent, and rows of no span mean nothing."""
        key = (S, L)
        t, M = self.torch, S * L
        f = dict(device="cuda", dtype=t.float32)
        scores = scores and not self.fused_attention(L)
        if key not in self._bufs:
            Mp = (M + 127) // 128 * 128  # fragment-major codes are read up to a multiple of 128 rows
            kp = (max(self.D, self.I) + 63) // 64 * 64  # the widest padded K of the layer's linears
            with self._on(stream):
                self._bufs = {key: dict(qkv=t.empty((M, self.W), **f), scores=t.empty(1, **f),
                                        ctx=t.empty((M, self.D), **f), out=t.empty((M, self.D), **f),
                                        inter=t.empty((M, self.I), **f), ffn=t.empty((M, self.D), **f),
                                        codes=t.empty(Mp * kp, device="cuda", dtype=t.int8),
                                        ascale=t.empty(M, **f))}
        b = self._bufs[key]
        if scores and b["scores"].numel() < S * self.H * L * L:  # beside the others, whose addresses a graph may hold
            with self._on(stream):
                b["scores"] = t.empty((S, self.H, L, L), **f)
        if t.cuda.is_current_stream_capturing() and not any(c is b for c in self._captured):
            self._captured.append(b)
        return b

    def _ints(self, name: str, t, shape) -> int:
        if t is None:
            return 0
        if t.dtype != self.torch.int32 or t.device.type != "cuda" or tuple(t.shape) != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 {list(shape)} tensor on the device")
        return t.data_ptr()

    def _floats(self, name: str, t, rows: int, more: bool = False) -> None:
        """Refuses what is no contiguous f32 [rows, D] device tensor; more: further rows may follow."""
        shape = tuple(t.shape)
        if len(shape) != 2 or shape[1] != self.D or not (shape[0] == rows or (more and shape[0] > rows)) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [{rows}, {self.D}] tensor, not {list(shape)}")
        if t.dtype != self.torch.float32 or t.device.type != "cuda":
            raise ValueError(f"{name} must be f32 on the device, not {t.dtype} on {t.device}")

    def forward(self, h, S: int, L: int, stream: int = 0, spans=None, pos=None, ids=None) -> None:
        """Runs every layer on h ([S*L, D] f32 on the device), in place, on `stream`. One shape's activations are
        kept, and until close() those of shapes that torch.cuda.graph captured: a call on another stream is ordered
        behind the last one's by the caller.

        spans (int32 [n, 2] on the device): the sequences are these spans of the S*L rows, first row and one past
        the last, ascending (enchip_attention_bias_dev; a list of a fixed number of them is filled up with S*L, S*L); what h holds in rows of none means nothing. pos (int32
        [S*L]): the rows' positions for `rope`, else row % L. ids (int32 [S*L]): the rows' adapters."""
        c, D, H, hd, M, W = self.ctx, self.D, self.H, self.hd, S * L, self.W
        self._floats("h", h, M)
        nspans = 0 if spans is None else spans.shape[0]
        d_spans, d_pos = self._ints("spans", spans, (nspans, 2)), self._ints("pos", pos, (M,))
        d_ids = self._ints("ids", ids, (M,))
        if ids is not None and self.adapters is None:
            raise ValueError("ids without adapters")
        kv = self.KV * hd
        b = self._buffers(S, L, stream, spans is None)
        qkv, scores, ctxv, out, inter, ffn = b["qkv"], b["scores"], b["ctx"], b["out"], b["inter"], b["ffn"]
        codes, ascale = b["codes"].data_ptr(), b["ascale"].data_ptr()
        q = qkv.data_ptr()
        scale = float(np.float32(1.0 / math.sqrt(hd)))  # encoder/attention.go:86

        def beside(li, name):  # the adapters of a linear, None without
            return self.adapters[li].get(name) if d_ids else None

        def route(w, low):  # the padded K when LN + quantization can run fused before w, else 0
            if not self.fuse_ln_quant or low is not None:
                return 0
            ok, ldq = c.frag_route(w, M)
            return ldq if ok and ldq <= D else 0

        def linear(name, w, x, bias, act, dst, low=None):  # one W8A8 linear on x [M, K]
            if low is not None:
                self._m(name + "+adapters")
                c.linear_adapters_dev(w, low, x.data_ptr(), M, d_ids, bias.data_ptr(), act, dst.data_ptr(), stream)
                return
            ok, ldq = c.frag_route(w, M)
            if ok:  # the kernels enchip_w8a8_linear_dev launches, as two timed calls
                self._m(name + ".quant")
                c.quant_rows_frag_dev(x.data_ptr(), M, w.K, codes, ldq, ascale, stream)
                self._m(name + ".gemm")
                c.pre_frag_dev(w, codes, ldq, M, ascale, bias.data_ptr(), act, dst.data_ptr(), stream)
            else:
                self._m(name)
                c.linear_dev(w, x.data_ptr(), M, bias.data_ptr(), act, dst.data_ptr(), stream)

        def ln_then(g, s_, y, nxt, label, low=None):  # h = LN(h + y); codes for weight nxt when it takes them
            ldq = route(nxt, low) if nxt is not None else 0
            self._m(label + ("+quant" if ldq else ""))
            if ldq:
                c.residual_layer_norm_quant_dev(h.data_ptr(), D, y.data_ptr(), D, M, D, g.data_ptr(), s_.data_ptr(),
                                                LN_EPS, codes, ldq, ascale, stream)
            else:
                c.residual_layer_norm_dev(h.data_ptr(), D, y.data_ptr(), D, M, D, g.data_ptr(), s_.data_ptr(), LN_EPS,
                                          stream)
            return ldq

        pending = 0  # padded K of codes already quantized for this layer's QKV
        for li, e in enumerate(self.handles):
            w, bias, act = e["qkv"]
            if pending:
                self._m("qkv.gemm")
                c.pre_frag_dev(w, codes, pending, M, ascale, bias.data_ptr(), act, q, stream)
            else:
                linear("qkv", w, h, bias, act, qkv, beside(li, "qkv"))
            if "q_norm" in e:
                self._m("head_norm")
                c.head_norm_rope_rows_dev(self.rope, self.rope_layout, q, W, q, W, S, L, H, self.KV, hd, e["q_norm"].data_ptr(),
                                          e["k_norm"].data_ptr(), self.norm_eps, d_pos, stream=stream)
            elif self.rope is not None:
                self._m("rope")
                c.rope_rows_dev(self.rope, self.rope_layout, q, W, q, W, S, L, H + self.KV, hd, d_pos, stream=stream)
            self._m("attention")
            if self.bias_attention(spans):
                c.attention_bias_dev(self.relpos, q, W, q + D * 4, W, q + (D + kv) * 4, W, ctxv.data_ptr(), D,
                                     S if spans is None else nspans, L if spans is None else M, H, self.KV, hd, scale, d_spans, stream)
            elif self.fused_attention(L):
                c.attention_f32_dev(q, q + D * 4, q + 2 * D * 4, 3 * D, ctxv.data_ptr(), D, S, L, H, hd, scale, stream)
            else:
                c.matmul_bt_f32_dev(q, 3 * D, q + D * 4, 3 * D, enchip.B_NK, scores.data_ptr(), L, L, hd, L,
                                    inner=(H, hd, hd, L * L), outer=(S, L * 3 * D, L * 3 * D, H * L * L),
                                    stream=stream)
                c.softmax_rows_scaled_dev(scores.data_ptr(), L, S * H * L, L, scale, stream)
                c.matmul_bt_f32_dev(scores.data_ptr(), L, q + 2 * D * 4, 3 * D, enchip.B_KN, ctxv.data_ptr(), D, L, L,
                                    hd, inner=(H, L * L, hd, hd), outer=(S, H * L * L, L * 3 * D, L * D),
                                    stream=stream)
            w, bias, act = e["o"]
            linear("o", w, ctxv, bias, act, out, beside(li, "o"))
            g, s = e["attn_ln"]
            w, bias, act = e["ffn_up"]
            if "ffn_gate" in e:
                wg, bg, act = e["ffn_gate"]
                ln_then(g, s, out, None, "attn_ln")
                self._m("ffn_gated")
                c.w8a8_gated_dev(wg, w, h.data_ptr(), M, bg.data_ptr(), bias.data_ptr(), act, inter.data_ptr(), stream)
                w, bias, act = e["ffn_down"]
                linear("ffn_down", w, inter, bias, act, ffn, beside(li, "ffn_down"))
                g, s = e["out_ln"]
                nxt = self.handles[li + 1]["qkv"][0] if li + 1 < len(self.handles) else None
                pending = ln_then(g, s, ffn, nxt, "out_ln", beside(li + 1, "qkv") if nxt is not None else None)
                continue
            up_low, down_low = beside(li, "ffn_up"), beside(li, "ffn_down")
            # adapters of FFN-down take the activations themselves
            gq = self.gelu_quant_route(act, e["ffn_down"][0], M) if down_low is None else 0
            up_act = enchip.ACT_NONE if gq else act
            ldq = ln_then(g, s, out, w, "attn_ln", up_low)
            if ldq:
                self._m("ffn_up.gemm")
                c.pre_frag_dev(w, codes, ldq, M, ascale, bias.data_ptr(), up_act, inter.data_ptr(), stream)
            else:
                linear("ffn_up", w, h, bias, up_act, inter, up_low)
            w, bias, act = e["ffn_down"]
            if gq:  # inter holds FFN-up's pre-activations: GELU them while quantizing
                self._m("ffn_down.gelu_quant")
                c.quant_rows_frag_gelu_dev(inter.data_ptr(), M, w.K, codes, gq, ascale, stream)
                self._m("ffn_down.gemm")
                c.pre_frag_dev(w, codes, gq, M, ascale, bias.data_ptr(), act, ffn.data_ptr(), stream)
            else:
                linear("ffn_down", w, inter, bias, act, ffn, down_low)
            g, s = e["out_ln"]
            nxt = self.handles[li + 1]["qkv"][0] if li + 1 < len(self.handles) else None
            pending = ln_then(g, s, ffn, nxt, "out_ln", beside(li + 1, "qkv") if nxt is not None else None)

    POOL_SPANS = 65535  # the most that one call pools

    def embed(self, h, S: int, L: int, pooled, stream: int = 0, spans=None, pos=None, ids=None) -> None:
        """forward(), then mean pooling + L2 normalisation of each sequence into pooled [S, D], or of
        each span into pooled [n, D] (rows of pooled past those stay as they were)."""
        self._floats("pooled", pooled, S if spans is None else spans.shape[0], more=True)
        self.forward(h, S, L, stream, spans, pos, ids)
        self._m("pool")
        if spans is not None:
            n = spans.shape[0]
            for z in range(0, n, self.POOL_SPANS):
                self.ctx.pool_mean_l2_spans_dev(h.data_ptr(), self.D, S * L, spans.data_ptr() + 8 * z, min(self.POOL_SPANS, n - z),
                                                self.D, pooled.data_ptr() + 4 * self.D * z, self.D, stream)
            self._m("end")
            return
        self.ctx.pool_mean_l2_dev(h.data_ptr(), self.D, S, L, self.D, pooled.data_ptr(), self.D, stream)
        self._m("end")

    def rerank(self, h, S: int, L: int, pooler, classifier, logits, stream: int = 0, ids=None) -> None:
        """forward(), then the cross-encoder head on each sequence's [CLS] row (row 0):
        logits [S, labels] = classifier(tanh(pooler(CLS))). pooler = (W [D, D], b [D]),
        classifier = (W [labels, D], b [labels]), f32 device tensors (PyTorch [out, in])."""
        c, D = self.ctx, self.D
        pw, pb = pooler
        cw, cb = classifier
        labels = cw.shape[0]
        if tuple(pw.shape) != (D, D) or tuple(cw.shape) != (labels, D) or tuple(logits.shape) != (S, labels):
            raise ValueError("rerank: pooler [D, D], classifier [labels, D], logits [S, labels]")
        self.forward(h, S, L, stream, ids=ids)
        self._m("head")
        b = self._bufs[(S, L)]
        if "pooled" not in b:
            with self._on(stream):
                b["pooled"] = self.torch.empty((S, D), device="cuda")
        pooled = b["pooled"]
        # CLS rows are every L-th row of h: pitch L*D
        c.matmul_bt_f32_dev(h.data_ptr(), L * D, pw.data_ptr(), D, enchip.B_NK, pooled.data_ptr(), D, S, D, D,
                            stream=stream)
        c.bias_act_rows_dev(pooled.data_ptr(), D, S, D, pb.data_ptr(), enchip.ACT_TANH, stream)
        c.matmul_bt_f32_dev(pooled.data_ptr(), D, cw.data_ptr(), D, enchip.B_NK, logits.data_ptr(), labels, S, D,
                            labels, stream=stream)
        c.bias_act_rows_dev(logits.data_ptr(), labels, S, labels, cb.data_ptr(), enchip.ACT_NONE, stream)
        self._m("end")
