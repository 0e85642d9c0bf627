// attention_bias.h -- attention with a learned relative position bias, over spans of rows.
//
// For query row i and key row j of one span, head h (key head h / (heads / kv_heads)):
//   out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = e^(scale q_i . k_j + b[j - i][h]),
// b by distance, clamped to reach rows either way. A span is [start, end) of the buffers' rows; rows of no
// span are neither read nor written. A query all of whose biases are -infinity gets zeros.
//
// The products, the split of operands into two f16 parts and the online softmax are attention_flash.h's:
// one workgroup takes 32 NW queries of one head and walks its keys in tiles of FA_KT, S^T = K Q^T and
// O^T = V^T P^T on v_mfma_f32_32x32x16_f16, three products per pair. Queries are scaled by scale log2 e before
// they are split, and the sums of the scores start at b log2 e, so a score leaves the MFMA in base 2 with its bias:
// the window of a tile's distances is staged in LDS beside its keys, and a lane reads its 16 from it (its queries are
// consecutive, so neighbouring lanes read neighbouring words).
//
// Bound by the products, 12 len^2 hd flops a head in three f16 parts, and by what stands between them (per score an
// exponential, a split into two parts, the maximum). Two blocks of 32 queries a wavefront give the products independent
// sums to run on and halve the loads of keys from LDS, where the registers allow it (heads of 32 and 64). On MI355X,
// flops of the formula (4 len^2 hd) a second: 64 x 512 rows of 12 heads of 64 183 us, 282 TF; 8192 rows 550 us, 375 TF
// (a third of a large f16 product's rate is 361); 20011 rows of documents of 1 to 1024, 16 heads of 128 that share 4 key
// heads, longest first 302 us, 270 TF. 1 x 512 rows take 12.3 us and 1 x 16 5.0, a call's latency. Values decide too: scores
// of twice the spread take up to 3% longer now that small weights hold bits, which the products' zeros had saved.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_flash.h"

#pragma clang fp contract(off)

namespace enchip {

// Weights are 2^(score - u) with a u below the running maximum, so that those far below it keep bits in f16's range: up
// to 2^AB_ABOVE when u is set, 2^15 at most (f16 ends at 65504), and off by 2^-25, f16's last place. A weight is held
// within 2^-22 of itself and 2^-36 (with AB_ABOVE) of the row's largest. u cancels in the division.
constexpr float AB_LAZY = 4.0f, AB_ABOVE = 15.0f - AB_LAZY;

// The u of a maximum m. Where m is so large that m - above is rounded to 16 below it, m itself.
__device__ __forceinline__ float ab_under(float m, float above) {
    const float u = m - above;
    return m - u > 15.5f ? m : u;
}

// Sums of long rows: the 16 weights of a lane's 32-key block are added in pairs, and what AB_FOLD keys gave is set aside
// (in the outputs' place, or LDS) and a new sum begun, so that roundings grow with AB_FOLD and not with the row. One sum
// over 131077 equal weights came out 8 10^-4 off, now 6 10^-6. 32768 rows of 12 heads of 64 8.86 ms, 8.77 in one sum; 8192 as before.
constexpr int AB_FOLD = 4096;

__device__ __forceinline__ float ab_sum16(const float (&x)[16]) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = x[e] + x[e + 8];
#pragma unroll
    for (int n = 4; n > 0; n /= 2)
#pragma unroll
        for (int e = 0; e < n; ++e) s[e] += s[e + n];
    return s[0];
}

struct AttnBias {
    const float *q, *k, *v;
    float *out;
    int64_t ldq, ldk, ldv, ldo;
    const int2 *spans;   // [nseq] start, end of ascending spans; null: nseq sequences of L rows
    const int4 *order;   // the spans longest first (attention_bias_order); null: as they come
    const float *table;  // [heads][2 reach + 1], b log2 e of distance -reach .. reach; null: no bias
    int nseq, heads, group, reach;
    int block0;  // with spans, the first of the launch's query blocks
    int L;       // rows of a sequence, or with spans those of the buffers
    int share;   // log2 of the heads of one key head that a workgroup takes, beside each other
    int parts;   // workgroups that split a query's keys
    float *part, *stat;  // parts > 1: [parts][rows][heads][hd] contexts, [parts][rows][heads][2] maxima and sums
    int64_t rows;        // of the buffers
    float scale;
};

// Key tiles of each of a sequence's parts.
__device__ __forceinline__ int ab_part_tiles(int nt, int parts) { return (nt + parts - 1) / parts; }

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
    static constexpr int WINDOW = 32 * NW * QPW + NW * FA_KT;  // most words of a tile's windows
    static constexpr int BIAS = 2 * Fa::STAGE;      // two windows behind the two stages
    static constexpr int STAT = BIAS + 2 * WINDOW * 4;  // a float2 a query, of what is set aside
    static constexpr int BYTES = STAT + 32 * NW * QPW * 8;
};

// The last of n things whose first(i), ascending, is at or below b, found 64 at a time by a wavefront; -1: none.
template <class F>
__device__ __forceinline__ int ab_last(int n, int b, F first) {
    const int lane = threadIdx.x & 63, count = n;
    for (int lo = 0;;) {
        const int step = (n + 63) / 64, z = lo + lane * step;
        const bool in = lane * step < n && first(min(z, count - 1)) <= b;
        const int below = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
        if (below == 0) return -1;
        n = min(step, n - (below - 1) * step);
        lo += (below - 1) * step;
        if (step == 1) return __builtin_amdgcn_readfirstlane(lo);
    }
}

// The workgroup's rows, QR = 2^qs queries from q0 on of the L from row0 on: false where it has none. Of ascending
// spans, span z has the query blocks start / QR + z .. of the call, at least as many as it needs. (Spans out of order
// leave queries out; nothing is read past the buffers.)
__device__ __forceinline__ bool ab_rows(const AttnBias &p, int b, int qs, int64_t &row0, int &len, int &q0) {
    if (p.spans == nullptr) {
        const int nqb = (p.L + (1 << qs) - 1) >> qs, z = b / nqb;
        row0 = (int64_t)z * p.L, len = p.L, q0 = (b - z * nqb) << qs;
        return true;
    }
    const int lo = ab_last(p.nseq, b, [&](int z) { return (max(p.spans[z].x, 0) >> qs) + z; });
    if (lo < 0) return false;
    const int2 s = p.spans[lo];
    const int start = min(max(s.x, 0), p.L), end = min(max(s.y, start), p.L);
    const int64_t at = (int64_t)(b - ((start >> qs) + lo)) << qs;
    if (at < 0 || at >= end - start) return false;
    row0 = start, len = end - start, q0 = (int)at;
    return true;
}

// The same of the launch's workgroup b in p.order: sequence by sequence, each head set's query blocks behind each other.
__device__ __forceinline__ bool ab_ordered(const AttnBias &p, int b, int qs, int &set, int64_t &row0, int &len, int &q0) {
    const int sets = p.heads >> p.share, lo = ab_last(p.nseq, b / sets, [&](int z) { return p.order[z].x; });
    if (lo < 0) return false;
    const int4 s = p.order[lo];
    const int at = b - s.x * sets, blocks = (s.z + (1 << qs) - 1) >> qs;
    if (at >= (int64_t)blocks * sets) return false;
    set = at / blocks;
    row0 = s.y, len = s.z, q0 = (at - set * blocks) << qs;
    return true;
}

// The spans by falling length, in steps of an eighth of a power of two of their key tiles, each with its first query
// block: a workgroup's time goes by its sequence's length, and a long one that starts last leaves the others waiting.
// Within a step the order is the atomics'; no result depends on it. One workgroup, at most AB_ORDER_MAX spans, which fill
// order whatever they hold (overlapping ones have more query blocks than the launch; those are left out).
constexpr int AB_ORDER_NT = 1024, AB_ORDER_MAX = 65536;
[[maybe_unused]] static __global__ __launch_bounds__(AB_ORDER_NT) void attention_bias_order(const int2 *__restrict__ spans, int nseq, int rows,
                                                                                           int qs, int4 *__restrict__ order) {
    constexpr int BINS = 256;  // steps of 2^24 tiles and less
    constexpr int COUNT = 44;  // a step's spans from bit 44 on, below them their query blocks: 2^25 of a span and less
    __shared__ unsigned long long next[BINS];
    const int tid = threadIdx.x;
    if (tid < BINS) next[tid] = 0;
    __syncthreads();
    auto span = [&](int z, int &start, int &len) {  // its step, longest first
        const int2 s = spans[z];
        start = min(max(s.x, 0), rows), len = min(max(s.y, start), rows) - start;
        const uint32_t f = __float_as_uint((float)(len / FA_KT + 1));
        return BINS - 1 - (int)((f >> 20) - (127u << 3));
    };
    for (int z = tid; z < nseq; z += AB_ORDER_NT) {
        int start, len;
        const int bin = span(z, start, len);
        atomicAdd(&next[bin], (1ull << COUNT) + (((unsigned)len + (1u << qs) - 1) >> qs));
    }
    __syncthreads();
    if (tid < 64) {
        unsigned long long own[BINS / 64], sum = 0;
#pragma unroll
        for (int i = 0; i < BINS / 64; ++i) own[i] = next[tid * (BINS / 64) + i], sum += own[i];
        unsigned long long at = sum;
        for (int o = 1; o < 64; o *= 2) {
            const unsigned long long v = __shfl_up(at, o, 64);
            if (tid >= o) at += v;
        }
        at -= sum;
#pragma unroll
        for (int i = 0; i < BINS / 64; ++i) next[tid * (BINS / 64) + i] = at, at += own[i];
    }
    __syncthreads();
    for (int z = tid; z < nseq; z += AB_ORDER_NT) {
        int start, len;
        const int bin = span(z, start, len);
        const unsigned long long at = atomicAdd(&next[bin], (1ull << COUNT) + (((unsigned)len + (1u << qs) - 1) >> qs));
        order[at >> COUNT] = make_int4((int)min(at & ((1ull << COUNT) - 1), 0x7fffffffull), start, len, 0);
    }
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

// A workgroup takes 32 NW QPW queries: QR = 32 NW QPW / 2^share rows of each of 2^share heads that have their keys in
// common, so that these are split once for all of them (and short sequences fill more of a workgroup).
// With parts > 1 the keys are split too, whole tiles to a part, and the contexts, not divided, go to scratch with their
// maxima and sums (attention_bias_join).
// A 1-D grid of (heads >> share) * parts * query blocks, XCD-aware (a sequence's query blocks of one head on one XCD),
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

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hf = lane >> 5;
    const int qs = __builtin_ctz(QB) - p.share, QR = 1 << qs;
    int set, part, L, q0;
    int64_t row0;
    if (p.order != nullptr) {
        // whole keys, the longest sequences of every head first, in runs of 4 blocks on one XCD (32768 rows of 64 equal
        // spans, 16 heads of 128 that share 4 key heads 473 us, runs of 1 498, of 8 466; 82 documents of 1 to 4096, 8 heads
        // 742, 757 and 754)
        part = 0;
        const int at = blockIdx.x;
        if (!ab_ordered(p, (at & ~31) + (at & 7) * 4 + ((at >> 3) & 3), qs, set, row0, L, q0)) return;
    } else {
        const int logical = xcd_logical_tile(blockIdx.x, gridDim.x), per_part = gridDim.x / ((p.heads >> p.share) * p.parts);
        const int sp = logical / per_part;
        set = sp / p.parts, part = sp - set * p.parts;
        if (!ab_rows(p, logical - sp * per_part + p.block0, qs, row0, L, q0)) return;
    }
    // the wavefront's head and its first query
    const int mate = (wave * 32 * QPW) >> qs, head = (set << p.share) + mate, qr = (wave * 32 * QPW) & (QR - 1), qw = q0 + qr;
    const bool active = qw < L;
    const int tiles = (L + FA_KT - 1) / FA_KT, per = ab_part_tiles(tiles, p.parts), tbeg = part * per, nt = min(tiles, tbeg + per);
    if (tbeg >= nt) return;
    const float *kbase = p.k + row0 * p.ldk + (head / p.group) * HD;
    const float *vbase = p.v + row0 * p.ldv + (head / p.group) * HD;
    // word w of a head's window: key kb0 + kk, query q0 + qi, w = kk - qi + QR - 1. A thread's words, as distances at
    // key 0 and places in the table.
    const int pitch = QR + FA_KT;
    int dist[WPT], place[WPT];
#pragma unroll
    for (int i = 0; i < WPT; ++i) {
        const int w = tid + NT * i, m = min(w / pitch, (1 << p.share) - 1);
        dist[i] = w - m * pitch - q0 - (QR - 1);
        place[i] = ((set << p.share) + m) * (2 * p.reach + 1) + p.reach;
    }
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
        if (p.table != nullptr)
#pragma unroll
            for (int i = 0; i < WPT; ++i) br[i] = p.table[place[i] + min(max(kb0 + dist[i], -p.reach), p.reach)];
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

    load_tile(tbeg);
#pragma unroll
    for (int u = 0; u < QPW; ++u)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) qt[u][b][i] *= c;
            ab_split8(qt[u][b], qh[u][b], ql[u][b]);
        }
    store_tile(tbeg & 1);
    lds_barrier();
    constexpr int FOLD = AB_FOLD / FA_KT;
    for (int t0 = tbeg;; t0 += FOLD) {
        for (int t = t0; t < min(nt, t0 + FOLD); ++t) {
            if (t + 1 < nt) load_tile(t + 1);
            if (active) {
                const char *khi = ab_lds + (t & 1) * Fa::STAGE, *klo = khi + Fa::KPLANE;
                const char *vhi = klo + Fa::KPLANE, *vlo = vhi + Fa::VPLANE;
                const float *window = reinterpret_cast<const float *>(ab_lds + Lay::BIAS) + (t & 1) * Lay::WINDOW + mate * pitch;
#pragma unroll
                for (int s = 0; s < FA_KT / 32; ++s) {
                    const int key0 = t * FA_KT + 32 * s;
                    if (key0 >= L) break;  // uniform: no barrier inside
                    // the scores' sums start at the bias; element e is key key0 + 4 hf + 8 (e / 4) + e % 4
                    f32x16 acc[QPW];
#pragma unroll
                    for (int u = 0; u < QPW; ++u) {
                        const float *bw = window + (32 * s + 4 * hf - (qr + 32 * u + r) + QR - 1);
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
                        // What is subtracted follows a query's running maximum only when that is AB_LAZY past where it was
                        // set: after the first tiles nothing is rescaled. (The difference of two numbers so near is exact.)
                        const bool up = mloc - m_run[u] > AB_ABOVE + AB_LAZY;
                        if (__builtin_amdgcn_ballot_w64(up) != 0) {
                            const float next = ab_under(mloc, AB_ABOVE), alpha = up ? __builtin_amdgcn_exp2f(m_run[u] - next) : 1.0f;
                            m_run[u] = up ? next : m_run[u];
                            l_run[u] *= alpha;
#pragma unroll
                            for (int i = 0; i < NOT; ++i)
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[u][i][e] *= alpha;
                        }
                        const float m_use = m_run[u] == -INFINITY ? 0.0f : m_run[u];  // nothing attended so far: every weight is 0
                        float x[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(acc[u][e] - m_use);
                        l_run[u] += ab_sum16(x);
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
        if (!active) {
            if (t0 + FOLD >= nt) return;
            continue;
        }
        const bool begun = t0 > tbeg, last = t0 + FOLD >= nt;
        int rr = r;
        asm volatile("" : "+v"(rr));  // the outputs' addresses are formed here, not held (and spilled) all along
        // the chunk's sums on top of what is set aside, which is in the outputs' place; divided after the last
#pragma unroll
        for (int u = 0; u < QPW; ++u) {
            const int query = qw + 32 * u + rr;
            float l_tot = l_run[u] + __shfl_xor(l_run[u], 32, 64), was = 0.0f;
            float2 *stat = reinterpret_cast<float2 *>(ab_lds + Lay::STAT) + (wave * QPW + u) * 32 + rr;
            if (begun) {
                was = __builtin_amdgcn_exp2f(stat->x - (m_run[u] == -INFINITY ? 0.0f : m_run[u]));
                l_tot += stat->y * was;
            }
            if (!last) *stat = make_float2(m_run[u], l_tot);  // by both halves of the lanes, the same
            if (query >= L) continue;
            float *orow = p.out + (row0 + query) * p.ldo + head * HD;
            float by = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
            if (p.parts > 1) {
                const int64_t at = (part * p.rows + row0 + query) * p.heads + head;
                orow = p.part + at * HD;
                if (last && hf == 0) *reinterpret_cast<float2 *>(p.stat + 2 * at) = make_float2(m_run[u], l_tot);
            }
            if (!last || p.parts > 1) by = 1.0f;
            if (begun) {
#pragma unroll
                for (int i = 0; i < NOT; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[u][i][e] += orow[32 * i + 8 * (e >> 2) + 4 * hf + (e & 3)] * was;
            }
#pragma unroll
            for (int i = 0; i < NOT; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x16 &a = o[u][i];
                    ab_store<VEC>(orow + 32 * i + 8 * g + 4 * hf,
                                  f32x4{a[4 * g] * by, a[4 * g + 1] * by, a[4 * g + 2] * by, a[4 * g + 3] * by});
                }
        }
        if (last) return;
#pragma unroll
        for (int u = 0; u < QPW; ++u) {
            l_run[u] = 0.0f;
#pragma unroll
            for (int i = 0; i < NOT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[u][i][e] = 0.0f;
        }
    }
}

// The parts of 32 rows of one head joined: out = sum_p o_p 2^(m_p - m) / sum_p l_p 2^(m_p - m).
template <int HD>
__global__ __launch_bounds__(256) void attention_bias_join(AttnBias p) {
    const int per_head = gridDim.x / p.heads, head = blockIdx.x / per_head;
    int64_t row0;
    int L, q0;
    if (!ab_rows(p, blockIdx.x - head * per_head, 5, row0, L, q0)) return;
    const int tiles = (L + FA_KT - 1) / FA_KT, per = ab_part_tiles(tiles, p.parts), parts = (tiles + per - 1) / per;
    for (int i = threadIdx.x; i < 32 * HD / 4; i += 256) {
        const int query = q0 + i / (HD / 4), col = 4 * (i % (HD / 4));
        if (query >= L) break;
        const int64_t at = (row0 + query) * p.heads + head, step = p.rows * p.heads;
        float m = -INFINITY, l = 0.0f;
        for (int u = 0; u < parts; ++u) m = fmaxf(m, p.stat[2 * (at + u * step)]);
        if (m == -INFINITY) m = 0.0f;
        f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int u = 0; u < parts; ++u) {
            const float2 st = *reinterpret_cast<const float2 *>(p.stat + 2 * (at + u * step));
            const f32x4 o = *reinterpret_cast<const f32x4 *>(p.part + (at + u * step) * HD + col);
            const float f = __builtin_amdgcn_exp2f(st.x - m);
            l += st.y * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] += o[e] * f;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float *to = p.out + (row0 + query) * p.ldo + head * HD + col;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = c[e] * inv;
    }
}

// Few queries: a workgroup takes 32 of one head and its NW wavefronts the head's keys, 32-key blocks w, w + NW, ...
// each with a softmax of its own; the NW maxima, sums and contexts meet in LDS. Nothing is shared before that, so
// keys and values go from memory straight to registers in the MFMA's order (a lane's value column is 8 loads of 4
// bytes, 32 lanes side by side), and there is no barrier in the loop: a call is a few memory round trips long. With
// NW = 1 it serves short sequences, many of them: no wavefront waits for another or is left without queries.
template <int HD, int NW>
struct AbSplit {
    static constexpr int PITCH = HD + 4;  // floats of a query's context: 8 of them start in distinct banks
    static constexpr int BYTES = NW * 32 * (PITCH + 2) * 4;
};

template <int HD, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attention_bias_split(AttnBias p) {
    using Lay = AbSplit<HD, NW>;
    constexpr int NB = HD / 16, NOT = HD / 32;
    extern __shared__ __attribute__((aligned(16))) char ab_lds[];
    float *ctx = reinterpret_cast<float *>(ab_lds), *top = ctx + NW * 32 * Lay::PITCH, *sum = top + NW * 32;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 31, hf = lane >> 5;
    int head, L, q0;
    int64_t row0;
    if (NW == 1 && p.order != nullptr) {
        const int at = blockIdx.x;
        if (!ab_ordered(p, (at & ~31) + (at & 7) * 4 + ((at >> 3) & 3), 5, head, row0, L, q0)) return;
    } else {
        const int logical = xcd_logical_tile(blockIdx.x, gridDim.x), per_head = gridDim.x / p.heads;
        head = logical / per_head;
        if (!ab_rows(p, logical - head * per_head + p.block0, 5, row0, L, q0)) return;
    }
    const float *kbase = p.k + row0 * p.ldk + (head / p.group) * HD;
    const float *vbase = p.v + row0 * p.ldv + (head / p.group) * HD;
    const float *table = p.table ? p.table + (int64_t)head * (2 * p.reach + 1) + p.reach : nullptr;
    const int ldk = (int)p.ldk, ldv = (int)p.ldv;
    f16x8 qh[NB], ql[NB];
    f32x16 o[NOT];
#pragma unroll
    for (int i = 0; i < NOT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;
    float qt[NB][8];
    {
        const float *qrow = p.q + (row0 + min(q0 + r, L - 1)) * p.ldq + head * HD;
#pragma unroll
        for (int b = 0; b < NB; ++b) load8(qrow + 16 * b + 8 * hf, qt[b]);
    }
    // heads of 128 load half of a key at a time, and 16 keys' values, for the registers
    constexpr bool AHEAD = HD < 128;
    auto split_q = [&] {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < 8; ++i) qt[b][i] *= p.scale * FA_LOG2E;
            ab_split8(qt[b], qh[b], ql[b]);
        }
    };
    if (!AHEAD) split_q();  // behind the first loads it would spill (551 documents of 1 to 200: 156 us for 126)
    int key0 = 32 * wave;
    for (bool begun = false;; begun = true) {
        const int stop = min(L, key0 + AB_FOLD * NW);
        for (; key0 < stop; key0 += 32 * NW) {
            const float *kt = kbase + (int64_t)key0 * ldk, *vt = vbase + (int64_t)key0 * ldv;
            const int last = L - 1 - key0;
            constexpr int KN = AHEAD ? NB : NB / 2, VN = AHEAD ? 2 : 1;
            float kx[KN][8], vx[NOT][VN][8];
            f32x16 acc;
            auto load_k = [&](int b0) {
#pragma unroll
                for (int b = 0; b < KN; ++b) load8(kt + (min(r, last) * ldk + 16 * (b0 + b) + 8 * hf), kx[b]);
            };
            load_k(0);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = key0 + 4 * hf + 8 * (e >> 2) + (e & 3) - (q0 + r);
                acc[e] = table != nullptr ? table[min(max(d, -p.reach), p.reach)] : 0.0f;
            }
            // value column 32 i + r: the eight keys at depth 8 hf .. of 16-key block kb
            auto load_v = [&](int kb) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float *row = vt + (min(16 * kb + 4 * hf + (j & 3) + 2 * (j & 4), last) * ldv + r);
#pragma unroll
                    for (int i = 0; i < NOT; ++i) vx[i][kb % VN][j] = row[32 * i];
                }
            };
            if (AHEAD) load_v(0), load_v(1);
            if (AHEAD && key0 == 32 * wave) split_q();
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b > 0 && b % KN == 0) load_k(b);
                f16x8 kh, kl;
                ab_split8(kx[b % KN], kh, kl);
                acc = mfma_split3(kh, kl, qh[b], ql[b], acc);
            }
            if (!AHEAD) load_v(0);
            if (key0 + 32 > L) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (8 * (e >> 2) + (e & 3) >= L - key0 - 4 * hf) acc[e] = -INFINITY;
            }
            float m = acc[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) m = fmaxf(m, acc[e]);
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            m = fmaxf(ab_under(m, 15.0f), m_run);  // followed at once: within 2^-40 of the row's largest weight
            const float m_use = m == -INFINITY ? 0.0f : m, alpha = __builtin_amdgcn_exp2f(m_run - m_use);
            m_run = m;
            l_run *= alpha;
#pragma unroll
            for (int i = 0; i < NOT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[i][e] *= alpha;
            float x[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(acc[e] - m_use);
            l_run += ab_sum16(x);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                f16x8 ph, pl;
                ab_split8(x + 8 * kb, ph, pl);
                if (!AHEAD && kb > 0) load_v(kb);
#pragma unroll
                for (int i = 0; i < NOT; ++i) {
                    f16x8 vh, vl;
                    ab_split8(vx[i][kb % VN], vh, vl);
                    o[i] = mfma_split3(vh, vl, ph, pl, o[i]);
                }
            }
        }
        l_run += __shfl_xor(l_run, 32, 64);
        // on top of what is set aside in LDS
        if (begun) {
            const float was = __builtin_amdgcn_exp2f(top[wave * 32 + r] - (m_run == -INFINITY ? 0.0f : m_run));
            l_run += sum[wave * 32 + r] * was;
#pragma unroll
            for (int i = 0; i < NOT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    o[i][e] += ctx[(wave * 32 + r) * Lay::PITCH + 32 * i + 8 * (e >> 2) + 4 * hf + (e & 3)] * was;
        }
        top[wave * 32 + r] = m_run, sum[wave * 32 + r] = l_run;  // by both halves of the lanes, the same
#pragma unroll
        for (int i = 0; i < NOT; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4 *>(ctx + (wave * 32 + r) * Lay::PITCH + 32 * i + 8 * g + 4 * hf) =
                    f32x4{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
        if (key0 >= L) break;
        l_run = 0.0f;
#pragma unroll
        for (int i = 0; i < NOT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    }
    __syncthreads();
    const int parts = min(NW, (L + 31) / 32);  // wavefronts that had keys
    for (int at = tid; at < 32 * HD / 4; at += 64 * NW) {
        const int query = at / (HD / 4), col = 4 * (at % (HD / 4));
        if (q0 + query >= L) break;
        float m = -INFINITY;
        for (int w = 0; w < parts; ++w) m = fmaxf(m, top[w * 32 + query]);
        if (m == -INFINITY) m = 0.0f;
        float l = 0.0f;
        f32x4 c = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < parts; ++w) {
            const float f = __builtin_amdgcn_exp2f(top[w * 32 + query] - m);
            l += sum[w * 32 + query] * f;
            const f32x4 part = *reinterpret_cast<const f32x4 *>(ctx + (w * 32 + query) * Lay::PITCH + col);
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] += part[e] * f;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float *to = p.out + (row0 + q0 + query) * p.ldo + head * HD + col;
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = c[e] * inv;
    }
}

}  // namespace enchip
