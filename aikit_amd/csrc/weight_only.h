// weight_only.h -- products of f32 activations with 4-bit weights of group scales, and gated
// pairs of products with 4-bit or int8 weights:
//   C[m, n] = sum_g s[n, g] sum_{k in g} A[m, k] q[n, k]                     (4-bit)
//   C[m, n] = act(y_gate[m, n] + bg[n]) * (y_up[m, n] + bu[n]),              (gated)
// y_i the product above, or for int8 weights ws[n] sum_k A[m, k] q[n, k]. The activations are
// never quantized, sums are f32.
//
// 4-bit image: [Np/64][Kp/32][64][16 B], 16 bytes per channel and 32 k: two codes a byte in k
// order, the lower k in the low half, in two's complement (the caller's c becomes q = c - 8);
// padding channels and k are 0. Np = N rounded up to 256, Kp = K rounded up to 64. Scales f16
// [Np/64][G][64], G = ceil(K / group). Int8 weights: the fragment-major image of kernels.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gated.h"
#include "gemm_q8w.h"
#include "kernels.h"

#pragma clang fp contract(off)

namespace enchip {

struct WoWeight {
    const int8_t *q;
    const void *s;  // _Float16 group scales (4-bit) or float channel scales (int8)
};

// The 4-bit image's 16 bytes of (channel n, chunk kc) of codes [N][ceil(K / 2)].
__global__ __launch_bounds__(256) void q4_image(const uint8_t *__restrict__ codes, uint4 *__restrict__ image, int N, int K,
                                                int chunks, int64_t total) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= total) return;
    const int64_t blk = t >> 6;
    const int64_t n = (blk / chunks) * 64 + (t & 63), kb = (K + 1) / 2;
    const int k0 = (int)(blk % chunks) * 32;
    uint32_t w[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        w[d] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int k = k0 + 8 * d + 2 * b;
            if (n >= N || k >= K) continue;
            uint32_t c = codes[n * kb + k / 2] ^ 0x88u;
            if (k + 1 >= K) c &= 0x0fu;
            w[d] |= c << (8 * b);
        }
    }
    image[t] = make_uint4(w[0], w[1], w[2], w[3]);
}

// scales [N][G] -> [Np/64][G][64], zero past N.
__global__ __launch_bounds__(256) void q4_scales(const uint16_t *__restrict__ s, uint16_t *__restrict__ out, int N, int G,
                                                 int64_t total) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= total) return;
    const int64_t n = (t >> 6) / G * 64 + (t & 63), g = (t >> 6) % G;
    out[t] = n < N ? s[n * G + g] : 0;
}

// Sum of v over the lanes of equal lane % 8, in all of them.
__device__ __forceinline__ float sum_units(float v) {
    v += __uint_as_float(lane_dpp<0x128>(__float_as_uint(v)));  // lane + 8 of the 16-lane row
    uint32_t a, b;
    lane_swap16(__float_as_uint(v), a, b);
    v = __uint_as_float(a) + __uint_as_float(b);
    lane_swap32(__float_as_uint(v), a, b);
    return __uint_as_float(a) + __uint_as_float(b);
}

// A few rows. A lane takes one channel and one unit of k at a time (16 bytes of weight: 32 k of a
// 4-bit one, 16 of an int8 one), a wavefront 8 channels x 8 units, a block of 256 or 128 k: eight
// whole cache lines. The block's activations reach the lanes through the wavefront's own LDS and
// stay in registers for all of its weights, so that a code costs its conversion and MB multiply-adds
// in f32. Of a workgroup's 8 wavefronts 1 << kbits split the blocks; the others take other channels,
// 8 NG each. One block ahead is in flight. The lanes' and the wavefronts' sums are added in one order.
//
// Bound by the reading of the weights while VALU work is short of it: per 4-bit KiB 32 codes a lane,
// 67 operations for one row and 33 more for each further one.
constexpr int WO_WAVES = 8;

template <int BITS, int MB, int NG, bool GATED>
__global__ __launch_bounds__(64 * WO_WAVES) void gemv_wo(const float *__restrict__ A, int64_t lda, WoWeight w0, WoWeight w1,
                                                         const float *__restrict__ b0, const float *__restrict__ b1, int act,
                                                         float *__restrict__ C, int64_t ldc, int M, int N, int K, int Kp,
                                                         FastDiv cpg, int G, int tilesN, int kbits) {
    constexpr int NW = GATED ? 2 : 1, CK = BITS == 4 ? 32 : 16, BK = 8 * CK, PU = CK + 4, LV = BK / 64;
    __shared__ __attribute__((aligned(16))) float s_a[WO_WAVES][MB][8 * PU];
    __shared__ float red[WO_WAVES][NG * NW * MB][8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, unit = lane >> 3, ch = lane & 7;
    const int ks = wave & ((1 << kbits) - 1), gsub = wave >> kbits, groups = NG * (WO_WAVES >> kbits);
    const int n0 = (blockIdx.x % tilesN) * 8 * groups, m0 = (blockIdx.x / tilesN) * MB, nw = n0 + 8 * NG * gsub;
    const int units = Kp / CK, blocks = (units + 7) / 8, step = 1 << kbits;
    const WoWeight w[2] = {w0, w1};
    const float *ar[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) ar[m] = A + (int64_t)min(m0 + m, M - 1) * lda;

    uint4 q[NG][NW];
    _Float16 sc[NG][NW];
    float av[MB][LV];
    auto load = [&](int blk) {
        const int u = min(8 * blk + unit, units - 1);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int n = nw + 8 * g;  // within Np: a multiple of 256
            const int64_t at = BITS == 4 ? ((int64_t)(n >> 6) * units + u) * 1024 + ((n & 63) + ch) * 16
                                         : ((int64_t)(n >> 5) * (units >> 1) + (u >> 1)) * 1024 + ((n & 31) + ch + 32 * (u & 1)) * 16;
#pragma unroll
            for (int t = 0; t < NW; ++t) {
                q[g][t] = *reinterpret_cast<const uint4 *>(w[t].q + at);
                if (BITS == 4)
                    sc[g][t] = static_cast<const _Float16 *>(
                        w[t].s)[((int64_t)(n >> 6) * G + min((int)cpg.div(u), G - 1)) * 64 + (n & 63) + ch];
            }
        }
        const int k = BK * blk + LV * lane;
#pragma unroll
        for (int m = 0; m < MB; ++m)
            if (k + LV <= K) {
#pragma unroll
                for (int e = 0; e < LV; ++e) av[m][e] = ar[m][k + e];
            } else {  // k past K counts as zero
#pragma unroll
                for (int e = 0; e < LV; ++e) {
                    const float x = ar[m][min(k + e, K - 1)];
                    av[m][e] = k + e < K ? x : 0.0f;
                }
            }
    };
    float sum[NG][NW][MB];
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int t = 0; t < NW; ++t)
#pragma unroll
            for (int m = 0; m < MB; ++m) sum[g][t][m] = 0.0f;
    if (ks < blocks) load(ks);
    for (int blk = ks; blk < blocks; blk += step) {
        float a[MB][CK];
        uint4 qc[NG][NW];
        float scc[NG][NW];
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int e = 0; e < LV; ++e) s_a[wave][m][(LV * lane / CK) * PU + LV * lane % CK + e] = av[m][e];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int t = 0; t < NW; ++t) qc[g][t] = q[g][t], scc[g][t] = BITS == 4 ? 16.0f * (float)sc[g][t] : 1.0f;
        if (blk + step < blocks) load(blk + step);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int e = 0; e < CK; e += 4) {
                const f32x4 v = *reinterpret_cast<const f32x4 *>(&s_a[wave][m][unit * PU + e]);
                a[m][e] = v.x, a[m][e + 1] = v.y, a[m][e + 2] = v.z, a[m][e + 3] = v.w;
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int t = 0; t < NW; ++t) {
                float y[MB];  // the unit's sums, unscaled
#pragma unroll
                for (int m = 0; m < MB; ++m) y[m] = 0.0f;
                const uint32_t qd[4] = {qc[g][t].x, qc[g][t].y, qc[g][t].z, qc[g][t].w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const uint32_t lo = qd[d];
                    if constexpr (BITS == 4) {
                        uint32_t hi = lo >> 4;
                        asm("" : "+v"(hi));  // one shift for its four codes
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const float f0 = __builtin_amdgcn_cvt_off_f32_i4((int)((lo >> (8 * b)) & 0xff));  // q / 16
                            const float f1 = __builtin_amdgcn_cvt_off_f32_i4((int)((hi >> (8 * b)) & 0xff));
#pragma unroll
                            for (int m = 0; m < MB; ++m)
                                y[m] = __builtin_fmaf(a[m][8 * d + 2 * b + 1], f1, __builtin_fmaf(a[m][8 * d + 2 * b], f0, y[m]));
                        }
                    } else {
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const float f = (float)(int8_t)((lo >> (8 * b)) & 0xff);
#pragma unroll
                            for (int m = 0; m < MB; ++m) y[m] = __builtin_fmaf(a[m][4 * d + b], f, y[m]);
                        }
                    }
                }
#pragma unroll
                for (int m = 0; m < MB; ++m)
                    sum[g][t][m] = BITS == 4 ? __builtin_fmaf(y[m], scc[g][t], sum[g][t][m]) : sum[g][t][m] + y[m];
            }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int t = 0; t < NW; ++t)
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                const float v = sum_units(sum[g][t][m]);
                if (lane < 8) red[wave][(g * NW + t) * MB + m][lane] = v;
            }
    __syncthreads();
    // thread: channel tid % (8 groups), row tid / (8 groups)
    const int chans = 8 * groups, c = tid & (chans - 1), m = tid / chans, n = n0 + c;
    if (m >= MB || m0 + m >= M || n >= N) return;
    const int g = (c >> 3) % NG, first = (c >> 3) / NG << kbits;
    float y[NW];
#pragma unroll
    for (int t = 0; t < NW; ++t) {
        y[t] = 0.0f;
        for (int j = 0; j < step; ++j) y[t] += red[first + j][(g * NW + t) * MB + m][c & 7];
        if (BITS == 8) y[t] *= static_cast<const float *>(w[t].s)[n];
    }
    float v = y[0];
    if constexpr (GATED) v = gate_f32(act, b0 ? y[0] + b0[n] : y[0], b1 ? y[1] + b1[n] : y[1]);
    C[(int64_t)(m0 + m) * ldc + n] = v;
}

// 8 codes of a 4-bit image word, in k order, as bf16 values q / 16 (exact).
__device__ __forceinline__ bf16x8 q4_widen8(uint32_t lo) {
    uint32_t hi = lo >> 4;
    asm("" : "+v"(hi));  // one shift for its four codes
    auto pair = [&](int b) {
        return q8w_pack(__float_as_uint(__builtin_amdgcn_cvt_off_f32_i4((int)((lo >> (8 * b)) & 0xff))),
                        __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4((int)((hi >> (8 * b)) & 0xff))));
    };
    return __builtin_bit_cast(bf16x8, (u32x4){pair(0), pair(1), pair(2), pair(3)});
}

// 8 int8 codes of a weight image, in k order, as bf16 values (exact).
__device__ __forceinline__ bf16x8 q8_widen8(uint32_t w0, uint32_t w1) {
    uint32_t x[4];
    q8w_widen4(w0, x[0], x[1]);
    q8w_widen4(w1, x[2], x[3]);
    return __builtin_bit_cast(bf16x8, (u32x4){x[0], x[1], x[2], x[3]});
}

// Tiles on the bf16 MFMA, activations split exactly into three bf16 parts (gemm_q8w.h). A
// workgroup computes 32 TM WM rows; each of its WM x WN x KS wavefronts TM x NT 32 x 32 tiles of
// products over its share of every K stage: NT channel blocks of one weight, or NT / 2 of each
// of the two, so a gate and its up projection meet in one lane. The stage's activations are split
// by all threads into three planes in LDS (double-buffered), the weights' codes go straight into
// registers and are widened there. A 4-bit weight's 32-deep chunk is summed from zero and added
// scaled: 16 multiply-adds for 6 MFMAs. The KS shares meet in LDS at the end, each wavefront
// finishing 16 / KS of the accumulator registers.
template <int BITS, bool GATED, int TM, int NT, int WM, int WN, int KS, int KC, bool VEC>
__global__ __launch_bounds__(64 * WM * WN * KS, 2) void gemm_wo(const float *__restrict__ A, int64_t lda, WoWeight w0,
                                                                WoWeight w1, const float *__restrict__ b0,
                                                                const float *__restrict__ b1, int act, float *__restrict__ C,
                                                                int64_t ldc, int M, int N, int K, int Kp, FastDiv cpg, int G,
                                                                int tilesN) {
    constexpr int NTHR = 64 * WM * WN * KS, BM = 32 * TM * WM, CPW = GATED ? 16 * NT : 32 * NT, BN = CPW * WN;
    constexpr int KB = KC / 32 / KS;  // chunks of a wavefront per stage
    constexpr int P = 2 * KC + 16, PL = BM * P, STAGE = 3 * PL;
    constexpr int LPR = KC / 4, AV = BM * LPR / NTHR, ER = 16 / KS;
    constexpr int RED = KS > 1 ? NTHR * (KS - 1) * ER * TM * NT * 4 : 0;
    constexpr int LDS = 2 * STAGE > RED ? 2 * STAGE : RED;
    static_assert(AV >= 1 && BM * LPR % NTHR == 0 && KB >= 1 && KC % (32 * KS) == 0 && 16 % KS == 0, "tile");
    static_assert(!GATED || NT % 2 == 0, "a tile of each weight");
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 31, hf = lane >> 5;
    const int logical = xcd_logical_tile(blockIdx.x, gridDim.x);
    const int m0 = (logical / tilesN) * BM, n0 = (logical % tilesN) * BN;
    const int ks = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
    const int lk = 4 * (tid % LPR), lr = tid / LPR;
    const WoWeight w[2] = {w0, w1};
    const float *ga[AV];
#pragma unroll
    for (int i = 0; i < AV; ++i) ga[i] = A + (int64_t)min(m0 + lr + (NTHR / LPR) * i, M - 1) * lda;
    const int nk32 = Kp / 32;
    // tile t: 32-channel block cb(t) of weight t % 2 (gated) or 0
    const int cb0 = (n0 + wn * CPW) >> 5;
    auto cb = [&](int t) { return cb0 + (GATED ? t >> 1 : t); };
    const int8_t *wb[NT];
    const _Float16 *sb[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const WoWeight &x = w[GATED ? t & 1 : 0];
        const int c = cb(t);
        wb[t] = x.q + (BITS == 4 ? (int64_t)(c >> 1) * nk32 * 1024 + ((c & 1) * 32 + r) * 16 + 8 * hf
                                 : (int64_t)c * nk32 * 1024 + lane * 16);
        sb[t] = static_cast<const _Float16 *>(x.s) + (BITS == 4 ? (int64_t)(c >> 1) * G * 64 + (c & 1) * 32 + r : 0);
    }
    f32x4 ra[AV];
    uint32_t wr[KB][NT][BITS / 2];
    _Float16 sc[KB][NT];
    auto load_a = [&](int c) {
        const int k = KC * c + lk;
        if (!VEC && KC * c + KC <= K) {  // uniform: all of the stage, in unaligned 16-byte loads
#pragma unroll
            for (int i = 0; i < AV; ++i) ra[i] = f32x4{ga[i][k], ga[i][k + 1], ga[i][k + 2], ga[i][k + 3]};
            return;
        }
#pragma unroll
        for (int i = 0; i < AV; ++i) {
            if (VEC) ra[i] = *reinterpret_cast<const f32x4 *>(ga[i] + min(k, K - 4));
            else
                ra[i] = f32x4{ga[i][min(k, K - 1)], ga[i][min(k + 1, K - 1)], ga[i][min(k + 2, K - 1)], ga[i][min(k + 3, K - 1)]};
        }
    };
    auto load_w = [&](int c) {
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const int kc = min(KC / 32 * c + KB * ks + b, nk32 - 1), g = BITS == 4 ? min((int)cpg.div(kc), G - 1) : 0;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (BITS == 4) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(wb[t] + (int64_t)kc * 1024);
                    wr[b][t][0] = v.x, wr[b][t][1] = v.y;
                    sc[b][t] = sb[t][(int64_t)g * 64];
                } else {
                    const uint4 v = *reinterpret_cast<const uint4 *>(wb[t] + (int64_t)kc * 1024);
                    wr[b][t][0] = v.x, wr[b][t][1] = v.y, wr[b][t][2] = v.z, wr[b][t][3] = v.w;
                }
            }
        }
    };
    auto store_a = [&](int c, char *st) {
        const int k = KC * c + lk;
#pragma unroll
        for (int i = 0; i < AV; ++i) {
            f32x4 v = ra[i];  // k past K counts as zero
            if (VEC) {
                if (k >= K) v = f32x4{0.f, 0.f, 0.f, 0.f};
            } else {
                v.x = k < K ? v.x : 0.f, v.y = k + 1 < K ? v.y : 0.f, v.z = k + 2 < K ? v.z : 0.f, v.w = k + 3 < K ? v.w : 0.f;
            }
            uint32_t a1[4], a2[4], a3[4];
            q8w_split3(v.x, a1[0], a2[0], a3[0]);
            q8w_split3(v.y, a1[1], a2[1], a3[1]);
            q8w_split3(v.z, a1[2], a2[2], a3[2]);
            q8w_split3(v.w, a1[3], a2[3], a3[3]);
            char *d = st + (lr + (NTHR / LPR) * i) * P + 2 * lk;
            *reinterpret_cast<uint2 *>(d) = make_uint2(q8w_pack(a1[0], a1[1]), q8w_pack(a1[2], a1[3]));
            *reinterpret_cast<uint2 *>(d + PL) = make_uint2(q8w_pack(a2[0], a2[1]), q8w_pack(a2[2], a2[3]));
            *reinterpret_cast<uint2 *>(d + 2 * PL) = make_uint2(q8w_pack(a3[0], a3[1]), q8w_pack(a3[2], a3[3]));
        }
    };
    f32x16 acc[TM][NT];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][t][e] = 0.0f;
    // Stage c + 1 is split into the other buffer behind stage c's MFMAs; past the last stage the
    // loads re-read it and the buffer is not used.
    const int nc = (Kp + KC - 1) / KC, last = nc - 1;
    load_a(0);
    load_w(0);
    store_a(0, lds);
    load_a(min(1, last));
    lds_barrier();
    for (int c = 0; c < nc; ++c) {
        const char *cur = lds + (c & 1) * STAGE;
        char *nxt = lds + ((c & 1) ^ 1) * STAGE;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            f32x16 part[TM][NT];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16x8 p[TM][3], q[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if constexpr (BITS == 4) q[t] = q4_widen8(wr[b][t][j]);
                    else q[t] = q8_widen8(wr[b][t][2 * j], wr[b][t][2 * j + 1]);
                }
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int x = 0; x < 3; ++x)
                        p[i][x] = *reinterpret_cast<const bf16x8 *>(cur + x * PL + (32 * (TM * wm + i) + r) * P +
                                                                    64 * (KB * ks + b) + 32 * hf + 16 * j);
#pragma unroll
                for (int x = 2; x >= 0; --x)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            f32x16 &s = BITS == 4 ? part[i][t] : acc[i][t];
                            if (BITS == 4 && j == 0 && x == 2) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) s[e] = 0.0f;
                            }
                            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[i][x], q[t], s, 0, 0, 0);
                        }
            }
            if (BITS == 4) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const float s = 16.0f * (float)sc[b][t];
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][t][e] = __builtin_fmaf(part[i][t][e], s, acc[i][t][e]);
                }
            }
        }
        load_w(min(c + 1, last));
        store_a(c + 1, nxt);
        load_a(min(c + 2, last));
        lds_barrier();
    }
    if constexpr (KS > 1) {
        // share s of the registers e in [ER s, ER s + ER) goes to wavefront s of the KS
        float *red = reinterpret_cast<float *>(lds);
        constexpr int PER = (KS - 1) * ER * TM * NT * 64;  // floats of one receiving wavefront
        const int mine = wave % (WM * WN);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s == ks) continue;
            float *d = red + (mine + WM * WN * s) * PER + (ks < s ? ks : ks - 1) * (ER * TM * NT * 64) + lane;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < ER; ++e) d[((i * NT + t) * ER + e) * 64] = acc[i][t][ER * s + e];
        }
        lds_barrier();
        const float *d = red + wave * PER + lane;
        // own registers first into the low places, then the others' shares in their order
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < ER; ++e) {
                    float v = 0.0f, o[KS];
#pragma unroll
                    for (int s = 0; s < KS; ++s) o[s] = acc[i][t][ER * s + e];
#pragma unroll
                    for (int s = 0; s < KS; ++s) v = ks == s ? o[s] : v;
#pragma unroll
                    for (int s = 0; s < KS - 1; ++s) v += d[s * (ER * TM * NT * 64) + ((i * NT + t) * ER + e) * 64];
                    acc[i][t][e] = v;
                }
    }
#pragma unroll
    for (int u = 0; u < (GATED ? NT / 2 : NT); ++u) {
        const int n = 32 * (cb0 + u) + r, nn = min(n, N - 1);
        float s[2], bb[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            s[x] = BITS == 8 ? static_cast<const float *>(w[x].s)[nn] : 1.0f;
            const float *b = x ? b1 : b0;
            bb[x] = GATED && b ? b[nn] : kNoBias;
        }
        if (n >= N) continue;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < ER; ++e) {
                const int m = m0 + 32 * (TM * wm + i) + acc_row(KS > 1 ? ER * ks + e : e, lane);
                float v = acc[i][GATED ? 2 * u : u][e] * s[0];
                if constexpr (GATED) v = gate_f32(act, v + bb[0], acc[i][2 * u + 1][e] * s[1] + bb[1]);
                if (m < M) C[(int64_t)m * ldc + n] = v;
            }
    }
}

}  // namespace enchip
