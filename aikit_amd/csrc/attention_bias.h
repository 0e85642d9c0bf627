// attention_bias.h -- attention with a learned relative position bias, over spans of rows.
//
// For query row i and key row j of one span, head h (key head h / (heads / kv_heads)):
//   out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = e^(scale q_i . k_j + b[j - i][h]),
// b by distance, clamped to reach rows either way. A span is [start, end) of the buffers' rows; rows of no
// span are neither read nor written. A query all of whose biases are -infinity gets zeros.
//
// The products, the split of operands into two f16 parts and the online softmax are attention_flash.h's:
// one workgroup takes 32 NW queries of one head and walks its keys in tiles of FA_KT, S^T = K Q^T and
// O^T = V^T P^T on v_mfma_f32_32x32x16_f16, three products per pair. The bias joins in base 2,
// y = fma(s, scale log2 e, b log2 e): the window of a tile's 32 NW + 63 distances is staged in LDS beside
// its keys, and a lane reads its 16 from it (its queries are consecutive, so neighbouring lanes read
// neighbouring words).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_flash.h"

#pragma clang fp contract(off)

namespace enchip {

constexpr float AB_LAZY = 8.0f;

struct AttnBias {
    const float *q, *k, *v;
    float *out;
    int64_t ldq, ldk, ldv, ldo;
    const int2 *spans;   // [nseq] start, end of ascending spans; null: nseq sequences of L rows
    const float *table;  // [heads][2 reach + 1], b log2 e of distance -reach .. reach; null: no bias
    int nseq, heads, group, reach;
    int blocks;  // with spans: query blocks of a head, L / (32 NW) + nseq
    int L;       // rows of a sequence, or with spans those of the buffers
    float scale;
};

// x less the low (high) half of h, exactly: one mixed fused multiply-add in place of a conversion and a subtraction.
__device__ __forceinline__ float ab_rest_lo(uint32_t h, float x) {
    float d;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(x));
    return d;
}
__device__ __forceinline__ float ab_rest_hi(uint32_t h, float x) {
    float d;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(h), "v"(x));
    return d;
}
// The parts of split_f16x8 and split_pair_f16 (attention_f32.h).
__device__ __forceinline__ void ab_pair(float a, float b, uint32_t &hw, uint32_t &lw) {
    hw = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
    lw = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){ab_rest_lo(hw, a), ab_rest_hi(hw, b)}, f16x2));
}
__device__ __forceinline__ void ab_split8(const float *x, f16x8 &hi, f16x8 &lo) {
    u32x4 h, l;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        uint32_t hw, lw;
        ab_pair(x[2 * s], x[2 * s + 1], hw, lw);
        h[s] = hw, l[s] = lw;
    }
    hi = __builtin_bit_cast(f16x8, h), lo = __builtin_bit_cast(f16x8, l);
}

template <int HD, int NW, int QPW>
struct AbLayout {
    using Fa = FaLayout<HD>;
    static constexpr int WINDOW = 32 * NW * QPW + FA_KT;  // distances of a tile (one to spare)
    static constexpr int BIAS = 2 * Fa::STAGE;      // two windows behind the two stages
    static constexpr int BYTES = BIAS + 2 * WINDOW * 4;
};

// The workgroup's rows: false where it has none. Of ascending spans, span z has the query blocks
// start / QB + z .. of the launch, at least as many as it needs; the last span whose first block is at or
// below b is found 64 at a time. (Spans out of order leave queries out; nothing is read past the buffers.)
template <int QB>
__device__ __forceinline__ bool ab_rows(const AttnBias &p, int b, int64_t &row0, int &len, int &q0) {
    if (p.spans == nullptr) {
        const int nqb = (p.L + QB - 1) / QB, z = b / nqb;
        row0 = (int64_t)z * p.L, len = p.L, q0 = (b - z * nqb) * QB;
        return true;
    }
    const int lane = threadIdx.x & 63;
    int lo = 0, n = p.nseq;
    for (;;) {
        const int step = (n + 63) / 64, z = lo + lane * step;
        const bool in = lane * step < n && max(p.spans[min(z, p.nseq - 1)].x, 0) / QB + z <= b;
        const int below = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
        if (below == 0) return false;
        n = min(step, n - (below - 1) * step);
        lo += (below - 1) * step;
        if (step == 1) break;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int2 s = p.spans[lo];
    const int start = min(max(s.x, 0), p.L), end = min(max(s.y, start), p.L);
    const int64_t at = (int64_t)(b - (start / QB + lo)) * QB;
    if (at < 0 || at >= end - start) return false;
    row0 = start, len = end - start, q0 = (int)at;
    return true;
}

// acc[u] += (ah + al) (b_h(u) + b_l(u)) less al b_l, a product of every accumulator in turn.
template <int N, class H, class Lo>
__device__ __forceinline__ void ab_mfma3(const f16x8 &ah, const f16x8 &al, H bh, Lo bl, f32x16 (&acc)[N]) {
#pragma unroll
    for (int u = 0; u < N; ++u) acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl(u), acc[u], 0, 0, 0);
#pragma unroll
    for (int u = 0; u < N; ++u) acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh(u), acc[u], 0, 0, 0);
#pragma unroll
    for (int u = 0; u < N; ++u) acc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh(u), acc[u], 0, 0, 0);
}

template <bool VEC>
__device__ __forceinline__ void ab_store(float *to, f32x4 v) {
    if constexpr (VEC) {
        *reinterpret_cast<f32x4 *>(to) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = v[i];
    }
}

// A 1-D grid of heads * query blocks, XCD-aware (a sequence's query blocks of one head on one XCD),
// AbLayout<HD, NW, QPW>::BYTES of dynamic LDS. q, k, v 16-byte aligned, their pitches multiples of 4 and at most
// INT32_MAX / FA_KT; VEC: ldo a multiple of 4 and out 16-byte aligned.
template <int HD, int NW, int QPW, bool VEC>
__global__ __launch_bounds__(64 * NW, HD == 128 || QPW == 2 ? 2 : 4) void attention_bias(AttnBias p) {
    using Fa = FaLayout<HD>;
    using Lay = AbLayout<HD, NW, QPW>;
    constexpr int NT = 64 * NW, QB = 32 * NW * QPW, WPT = (Lay::WINDOW + NT - 1) / NT;
    constexpr int NB = HD / 16, NOT = HD / 32;
    constexpr int KCH = FA_KT * HD / 8, VCH = (FA_KT / 2) * HD / 4;
    constexpr int KPT = (KCH + NT - 1) / NT, VPT = (VCH + NT - 1) / NT;
    using Ops = SplitOps<true>;
    using vec8 = typename Ops::vec8;
    extern __shared__ __attribute__((aligned(16))) char ab_lds[];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, hf = lane >> 5;
    const int logical = xcd_logical_tile(blockIdx.x, gridDim.x), per_head = gridDim.x / p.heads;
    const int head = logical / per_head;
    int64_t row0;
    int L, q0;
    if (!ab_rows<QB>(p, logical - head * per_head, row0, L, q0)) return;
    const int qw = q0 + 32 * QPW * wave;  // the wavefront's first query
    const bool active = qw < L;
    const int nt = (L + FA_KT - 1) / FA_KT;
    const float *kbase = p.k + row0 * p.ldk + (head / p.group) * HD;
    const float *vbase = p.v + row0 * p.ldv + (head / p.group) * HD;
    const float *table = p.table ? p.table + (int64_t)head * (2 * p.reach + 1) + p.reach : nullptr;
    const float c = p.scale * FA_LOG2E;  // of the queries: scores come out in base 2

    vec8 qh[QPW][NB], ql[QPW][NB];
    float qt[QPW][NB][8];
#pragma unroll
    for (int u = 0; u < QPW; ++u) {
        const float *qrow = p.q + (row0 + min(qw + 32 * u + r, L - 1)) * p.ldq + head * HD;
#pragma unroll
        for (int b = 0; b < NB; ++b) load8(qrow + 16 * b + 8 * hf, qt[u][b]);
    }
    f32x4 kr[KPT][2], vr[VPT][2];
    float br[WPT] = {};
    const int ldk = (int)p.ldk, ldv = (int)p.ldv;
    auto load_tile = [&](int t) {
        const int kb0 = t * FA_KT, klast = L - 1 - kb0;
        const float *kt = kbase + (int64_t)kb0 * ldk, *vt = vbase + (int64_t)kb0 * ldv;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int ch = tid + NT * i;
            if (ch < KCH) {
                const float *at = kt + (min(ch / (HD / 8), klast) * ldk + (ch % (HD / 8)) * 8);
                kr[i][0] = *reinterpret_cast<const f32x4 *>(at);
                kr[i][1] = *reinterpret_cast<const f32x4 *>(at + 4);
            }
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int ch = tid + NT * i;
            if (ch < VCH) {
                const int pr = ch / (HD / 4), col = (ch % (HD / 4)) * 4;
                vr[i][0] = *reinterpret_cast<const f32x4 *>(vt + (min(2 * pr, klast) * ldv + col));
                vr[i][1] = *reinterpret_cast<const f32x4 *>(vt + (min(2 * pr + 1, klast) * ldv + col));
            }
        }
        // word w of the window: key kb0 + kk, query q0 + qi, w = kk - qi + QB - 1
        if (table != nullptr)
#pragma unroll
            for (int i = 0; i < WPT; ++i) br[i] = table[min(max(kb0 - q0 - (QB - 1) + tid + NT * i, -p.reach), p.reach)];
    };
    auto store_tile = [&](int s) {
        char *khi = ab_lds + s * Fa::STAGE, *klo = khi + Fa::KPLANE;
        char *vhi = klo + Fa::KPLANE, *vlo = vhi + Fa::VPLANE;
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int ch = tid + NT * i;
            if (ch < KCH) {
                const int key = ch / (HD / 8), col = (ch % (HD / 8)) * 8;
                const float x[8] = {kr[i][0].x, kr[i][0].y, kr[i][0].z, kr[i][0].w,
                                    kr[i][1].x, kr[i][1].y, kr[i][1].z, kr[i][1].w};
                vec8 h, l;
                ab_split8(x, h, l);
                *reinterpret_cast<vec8 *>(khi + key * Fa::KP + 2 * col) = h;
                *reinterpret_cast<vec8 *>(klo + key * Fa::KP + 2 * col) = l;
            }
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int ch = tid + NT * i;
            if (ch < VCH) {
                const int pr = ch / (HD / 4), col = (ch % (HD / 4)) * 4;
                const int kk = 2 * pr, pos = (kk & ~15) | fa_perm16(kk & 15);
                const float a[4] = {vr[i][0].x, vr[i][0].y, vr[i][0].z, vr[i][0].w};
                const float b[4] = {vr[i][1].x, vr[i][1].y, vr[i][1].z, vr[i][1].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t hw, lw;
                    ab_pair(a[j], b[j], hw, lw);
                    const int vo = (col + j) * Fa::VP + ((2 * pos) ^ fa_vswz(col + j));
                    *reinterpret_cast<uint32_t *>(vhi + vo) = hw;
                    *reinterpret_cast<uint32_t *>(vlo + vo) = lw;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < WPT; ++i)
            if (tid + NT * i < Lay::WINDOW) reinterpret_cast<float *>(ab_lds + Lay::BIAS)[s * Lay::WINDOW + tid + NT * i] = br[i];
    };

    f32x16 o[QPW][NOT];
    float m_run[QPW], l_run[QPW];
#pragma unroll
    for (int u = 0; u < QPW; ++u) {
#pragma unroll
        for (int i = 0; i < NOT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[u][i][e] = 0.0f;
        m_run[u] = -INFINITY, l_run[u] = 0.0f;
    }

    load_tile(0);
#pragma unroll
    for (int u = 0; u < QPW; ++u)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) qt[u][b][i] *= c;
            ab_split8(qt[u][b], qh[u][b], ql[u][b]);
        }
    store_tile(0);
    lds_barrier();
    for (int t = 0; t < nt; ++t) {
        if (t + 1 < nt) load_tile(t + 1);
        if (active) {
            const char *khi = ab_lds + (t & 1) * Fa::STAGE, *klo = khi + Fa::KPLANE;
            const char *vhi = klo + Fa::KPLANE, *vlo = vhi + Fa::VPLANE;
            const float *window = reinterpret_cast<const float *>(ab_lds + Lay::BIAS) + (t & 1) * Lay::WINDOW;
#pragma unroll
            for (int s = 0; s < FA_KT / 32; ++s) {
                const int key0 = t * FA_KT + 32 * s;
                if (key0 >= L) break;  // uniform: no barrier inside
                // the scores' sums start at the bias; element e is key key0 + 4 hf + 8 (e / 4) + e % 4
                f32x16 acc[QPW];
#pragma unroll
                for (int u = 0; u < QPW; ++u) {
                    const float *bw = window + (32 * s + 4 * hf - (32 * (QPW * wave + u) + r) + QB - 1);
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[u][e] = bw[8 * (e >> 2) + (e & 3)];
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const int off = (32 * s + r) * Fa::KP + 2 * (16 * b + 8 * hf);
                    const vec8 kh = *reinterpret_cast<const vec8 *>(khi + off);
                    const vec8 kl = *reinterpret_cast<const vec8 *>(klo + off);
                    ab_mfma3<QPW>(kh, kl, [&](int u) { return qh[u][b]; }, [&](int u) { return ql[u][b]; }, acc);
                }
                vec8 ph[QPW][2], pl[QPW][2];
#pragma unroll
                for (int u = 0; u < QPW; ++u) {
                    const int lim = L - key0 - 4 * hf;
                    if (__builtin_expect(key0 + 32 > L, 0)) {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (8 * (e >> 2) + (e & 3) >= lim) acc[u][e] = -INFINITY;
                    }
                    float mloc = acc[u][0];
#pragma unroll
                    for (int e = 1; e < 16; ++e) mloc = fmaxf(mloc, acc[u][e]);
                    {
                        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mloc), __float_as_uint(mloc), false, false);
                        mloc = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
                    }
                    // The subtracted maximum follows a query's running maximum only when that is AB_LAZY above it:
                    // weights up to 2^AB_LAZY keep their precision, and after the first tiles nothing is rescaled.
                    const bool up = mloc > m_run[u] + AB_LAZY;
                    if (__builtin_amdgcn_ballot_w64(up) != 0) {
                        const float alpha = up ? __builtin_amdgcn_exp2f(m_run[u] - mloc) : 1.0f;
                        m_run[u] = up ? mloc : m_run[u];
                        l_run[u] *= alpha;
#pragma unroll
                        for (int i = 0; i < NOT; ++i)
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[u][i][e] *= alpha;
                    }
                    const float m_use = m_run[u] == -INFINITY ? 0.0f : m_run[u];  // nothing attended so far: every weight is 0
                    float x[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        x[e] = __builtin_amdgcn_exp2f(acc[u][e] - m_use);
                        l_run[u] += x[e];
                    }
                    ab_split8(x, ph[u][0], pl[u][0]);
                    ab_split8(x + 8, ph[u][1], pl[u][1]);
                }
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int i = 0; i < NOT; ++i) {
                        const int off = (32 * i + r) * Fa::VP + 64 * s + 32 * (kb ^ (i & 1)) + 16 * (hf ^ (r >> 4));
                        const vec8 vh = *reinterpret_cast<const vec8 *>(vhi + off);
                        const vec8 vl = *reinterpret_cast<const vec8 *>(vlo + off);
                        f32x16 d[QPW];
#pragma unroll
                        for (int u = 0; u < QPW; ++u) d[u] = o[u][i];
                        ab_mfma3<QPW>(vh, vl, [&](int u) { return ph[u][kb]; }, [&](int u) { return pl[u][kb]; }, d);
#pragma unroll
                        for (int u = 0; u < QPW; ++u) o[u][i] = d[u];
                    }
                }
                __builtin_amdgcn_s_setprio(0);
            }
        }
        if (t + 1 < nt) store_tile((t + 1) & 1);
        lds_barrier();
    }

    if (!active) return;
#pragma unroll
    for (int u = 0; u < QPW; ++u) {
        const float l_tot = l_run[u] + __shfl_xor(l_run[u], 32, 64);
        const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
        const int query = qw + 32 * u + r;
        if (query >= L) continue;
        float *orow = p.out + (row0 + query) * p.ldo + head * HD;
#pragma unroll
        for (int i = 0; i < NOT; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x16 &a = o[u][i];
                ab_store<VEC>(orow + 32 * i + 8 * g + 4 * hf,
                              f32x4{a[4 * g] * inv, a[4 * g + 1] * inv, a[4 * g + 2] * inv, a[4 * g + 3] * inv});
            }
    }
}

}  // namespace enchip
