// weight_only.h -- products of f32 activations with 4-bit weights of group scales, and gated
// pairs of products with 4-bit or int8 weights:
//   C[m, n] = sum_g s[n, g] sum_{k in g} A[m, k] q[n, k]                     (4-bit)
//   C[m, n] = act(y_gate[m, n] + bg[n]) * (y_up[m, n] + bu[n]),              (gated)
// y_i the product above, or for int8 weights ws[n] sum_k A[m, k] q[n, k]. The activations are
// never quantized, sums are f32.
//
// 4-bit image: [Np/64][Kp/32][64][16 B], 16 bytes per channel and 32 k, codes c = q + 8. A word holds
// 8 k's: k 2i in bits 4i .. and k 2i + 1 in bits 16 + 4i .., so that one mask and one packed f16
// subtraction give two neighbouring values. Padding channels and k are 0 (c = 8). Np = N rounded up
// to 256, Kp = K rounded up to 64. Scales f16 [Np/64][G][64], G = ceil(K / group). Int8 weights: the
// fragment-major image of kernels.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_f32.h"
#include "gated.h"
#include "gemm_f32.h"
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
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + 8 * d + 2 * i;
            uint32_t c = n < N && k < K ? codes[n * kb + k / 2] : 0x88u;
            if (k + 1 >= K) c = (c & 0x0fu) | 0x80u;
            w[d] |= (c & 15u) << (4 * i) | (c >> 4) << (16 + 4 * i);
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

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// 8 neighbouring codes as four pairs of f16 values, exactly: a code in the low bits of 1024 (f16's
// step there is 1), less 1024 and the code's offset. Conversions to f32 take four times a plain
// operation's issue; these take one each for two codes.
__device__ __forceinline__ void widen8_q4(uint32_t w, f16x2 (&h)[4]) {
    uint32_t low = 0x000f000fu, high = 0x00f000f0u, base = 0x64006400u;
    asm("" : "+s"(low), "+s"(high));  // kept in registers: one v_and_or each
    asm("" : "+v"(base));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = w >> (8 * i);
        h[2 * i] = __builtin_bit_cast(f16x2, (v & low) | base) - f16x2{(_Float16)1032.0f, (_Float16)1032.0f};
        // four bits up a code counts 16: (1024 + 16 c) / 16 - 72, exactly, for a shift less
        h[2 * i + 1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (v & high) | base),
                                                 f16x2{(_Float16)0.0625f, (_Float16)0.0625f},
                                                 f16x2{(_Float16)-72.0f, (_Float16)-72.0f});
    }
}
__device__ __forceinline__ void widen8_q8(uint32_t w0, uint32_t w1, f16x2 (&h)[4]) {
    const uint32_t w[2] = {w0 ^ 0x80808080u, w1 ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w[i >> 1], i & 1 ? 0x04030402u : 0x04010400u)) -
               f16x2{(_Float16)1152.0f, (_Float16)1152.0f};
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
// MI355X, us: 4 bits, 8192 x 8192, 1 row 8.4 to 10 (34.6 MB, 4 TB/s; its vector instructions issue for 6),
// 2 rows 13.0, 4 rows 17.8; K = N = 4096 1 row 5.3, 4 rows 7.8; the gated pair of K = 1024, N = 4096 4.4 (4
// bits) and 4.8 (int8): one trip to memory and the launch. A lane on a channel's 16 bytes with its activations
// read from LDS for every weight took 15.9 (2 rows) and 26.2 (4 rows) of 8192 x 8192. NG = 2 where it leaves
// two workgroups a CU, so that a block's activations serve two groups of channels.
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
                    if constexpr (BITS == 4) {
                        // a byte's low and high halves, as q / 16: k 0, 4, 1, 5 and 2, 6, 3, 7 of the word's 8
                        const uint32_t lo = qd[d] ^ 0x88888888u;
                        uint32_t hi = lo >> 4;
                        asm("" : "+v"(hi));  // one shift for its four codes
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const float f0 = __builtin_amdgcn_cvt_off_f32_i4((int)((lo >> (8 * b)) & 0xff));
                            const float f1 = __builtin_amdgcn_cvt_off_f32_i4((int)((hi >> (8 * b)) & 0xff));
                            const int k = 8 * d + (b >> 1) + 4 * (b & 1);
#pragma unroll
                            for (int m = 0; m < MB; ++m)
                                y[m] = __builtin_fmaf(a[m][k + 2], f1, __builtin_fmaf(a[m][k], f0, y[m]));
                        }
                    } else {
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const float f = (float)(int8_t)((qd[d] >> (8 * b)) & 0xff);
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

// More rows run on the f16 MFMA. split_rows scales each row of activations by the power of two that
// brings its largest to 2^14 .. 2^15 and splits it into two f16 parts: hi, rounded to f16's 11 bits, and lo, what
// is left times 2^12, rounded to 11 again. What is left is at most half of hi's step, so lo errs by at most
// 2^-23 of the activation (f32's own step; what is left is a multiple of that step, so three of four
// activations are exact). lo at hi's own scale would run into f16's smallest step and keep 2^-39 of
// the row's largest: nothing of an activation that far below it. Codes are f16 values exactly, and so are
// codes / 2^12, which lo is multiplied with: products are exact and two MFMAs stand for one in f32. Where hi is
// subnormal (under 2^-14 scaled, 2^-28 to 2^-29 of the row's largest) it has fewer bits: a row's block of 128 k
// with such an activation is marked: its parts are 0, and the products add it on the f32 MFMA at their end. MI355X,
// 4 bits, 4096 rows of K = N = 4096: 280 us for normal activations, 281 behind a GELU, 334 with one of 1000 a
// thousand times larger, 2230 where every block is marked (softmax rows).
//
// Parts, in the A operand's order for the weights' order of k: [M/32][Ka/32] x 4 KiB, plane x and
// step j of chunk kc at x 2048 + j 1024, 16 bytes per lane: row lane % 32, k = 32 kc + 16 (lane / 32) + 8 j
// .. + 7. Ka = K rounded up to 128, zero past K. Rows past M are not written (and no output is theirs).
//
// Two parts take two thirds of the MFMAs of three exact bf16 parts, made in every tile that reads the row:
// those took 57.9 us for 512 rows of K = N = 4096 in 4 bits where this takes 50 to 53, 436 where it takes 272
// to 280 for 4096. lo's own codes cost 1 to 3% of that (a packed multiplication for two of them). A row costs 8 bytes an
// element, read and written once: MI355X 4096 x 4096 30 to 35 us (4 TB/s), 512 x 1024 3.1 to 4.1 us and 32 x
// 4096 3.7 (a launch and one pass through a row). Neighbouring rows, whose 16-byte pieces share lines, run on one
// die: 4096 x 8192 84 us, on different ones 131.
struct SplitRows {
    const char *parts;
    const float2 *scale;   // [M] the row's power of two, negative for a row with marks, and the one that takes it back
    const uint8_t *mark;   // [M/32][Ka/128][32]
};
typedef float f32x2v __attribute__((ext_vector_type(2)));
constexpr int SPLIT_WAVES = 4;
constexpr float LO = 4096.0f;  // what lo is scaled by

// The codes that lo's parts are multiplied with: q / 2^12, exact and normal in f16 for |q| from 1 to 128.
__device__ __forceinline__ f16x8 lo_codes(const f16x8 &q) { return q * (_Float16)(1.0f / LO); }

// WPR wavefronts per row, thread t of them holding CH granules of 8 k at a time, 64 WPR apart. HELD: all of
// the row's (K <= 512 WPR CH), read once. Otherwise the row is read twice.
template <int WPR, int CH, bool HELD, bool VEC>
__global__ __launch_bounds__(64 * SPLIT_WAVES) void split_rows(const float *__restrict__ A, int64_t lda, char *__restrict__ parts,
                                                               float2 *__restrict__ scale, uint8_t *__restrict__ mark, int M,
                                                               int K, int nkc) {
    constexpr int NT = 64 * WPR;
    static_assert(WPR == 1 || WPR == SPLIT_WAVES, "a wavefront or a workgroup per row");
    __shared__ float s_m[SPLIT_WAVES];
    __shared__ int s_mark[SPLIT_WAVES];
    const int t = threadIdx.x & (NT - 1), wave = threadIdx.x >> 6;
    const int b = xcd_logical_tile(blockIdx.x, gridDim.x), row = WPR == 1 ? b * SPLIT_WAVES + wave : b;
    if (row >= M) return;  // WPR 1 only: no barrier there
    const float *a = A + (int64_t)row * lda;
    const int granules = 4 * nkc, rounds = HELD ? 1 : (granules + NT * CH - 1) / (NT * CH);
    f32x4 v[CH][2];
    auto load = [&](int i, f32x4 (&x)[2]) {
        const int k = 8 * (t + NT * i);
        if (VEC) {
            x[0] = *reinterpret_cast<const f32x4 *>(a + min(k, K - 4));
            x[1] = *reinterpret_cast<const f32x4 *>(a + min(k + 4, K - 4));
            if (k >= K) x[0] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (k + 4 >= K) x[1] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = a[min(k + e, K - 1)];
                x[e >> 2][e & 3] = k + e < K ? t : 0.0f;
            }
        }
    };
    float m = 0.0f;
    auto largest = [&](const f32x4 (&x)[2]) {  // fmaxf passes NaN over
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[e >> 2][e & 3]));
    };
    for (int c = 0; c < rounds; ++c) {
#pragma unroll
        for (int i = 0; i < CH; ++i) load(c * CH + i, v[i]);
#pragma unroll
        for (int i = 0; i < CH; ++i) largest(v[i]);
    }
    m = wave_absmax(m);
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) s_m[wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; ++w) m = fmaxf(m, s_m[w]);
    }
    // m in [2^(E-127), 2^(E-126)): times 2^(141-E), at most 2^127; an infinite m (E = 255) keeps infinities
    // and makes the finite values beside them small
    const int E = (int)(__float_as_uint(m) >> 23), F = min(268 - E, 254);
    const float up = __uint_as_float((uint32_t)F << 23);
    uint64_t marked = 0;
    auto store = [&](int i, f32x4 (&x)[2]) {
        const int g = t + NT * i;
        uint32_t hi[4], lo[4];
        bool small = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p = x[e >> 1][2 * (e & 1)] * up, q = x[e >> 1][2 * (e & 1) + 1] * up;
            const f16x2 h = __builtin_convertvector(f32x2v{p, q}, f16x2);
            const f32x2v l = {__builtin_fmaf((float)h.x, -LO, p * LO), __builtin_fmaf((float)h.y, -LO, q * LO)};  // exact
            hi[e] = __builtin_bit_cast(uint32_t, h);
            lo[e] = E == 255 ? 0u : __builtin_bit_cast(uint32_t, __builtin_convertvector(l, f16x2));  // inf - inf
            small |= (p != 0.0f && fabsf(p) < 0x1p-14f) || (q != 0.0f && fabsf(q) < 0x1p-14f);
        }
        // a block's 16 granules are a 16-lane row
        const uint64_t smalls = E == 255 ? 0 : __builtin_amdgcn_ballot_w64(small);
        const bool mk = (smalls >> (threadIdx.x & 48) & 0xffffu) != 0;
        marked |= smalls;
        if (g >= granules) return;
        char *d = parts + ((int64_t)(row >> 5) * nkc + (g >> 2)) * 4096 + (g & 1) * 1024 + ((row & 31) + 32 * ((g >> 1) & 1)) * 16;
        *reinterpret_cast<uint4 *>(d) = mk ? make_uint4(0, 0, 0, 0) : make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(d + 2048) = mk ? make_uint4(0, 0, 0, 0) : make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if ((g & 15) == 0) mark[((int64_t)(row >> 5) * (nkc >> 2) + (g >> 4)) * 32 + (row & 31)] = mk;
    };
    for (int c = 0; c < rounds; ++c) {
        if constexpr (!HELD) {
#pragma unroll
            for (int i = 0; i < CH; ++i) load(c * CH + i, v[i]);
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) store(c * CH + i, v[i]);
    }
    bool some_marked = marked != 0;
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) s_mark[wave] = some_marked;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; ++w) some_marked |= s_mark[w] != 0;
    }
    if (t == 0)
        scale[row] = make_float2(some_marked ? -up : up, __uint_as_float(F == 254 ? 0x400000u : (uint32_t)(254 - F) << 23));
}

// What a product of split rows reads besides the weights.
struct WoRows {
    SplitRows a;
    const float *A;  // the rows as they are, for marked blocks
    int64_t lda;
    int M, N, K, Kp, nkc, G;
    FastDiv cpg;
};

// TM x NT tiles' weights of one wavefront: NT channel blocks of one weight, or NT / 2 of each of the
// two, so that a gate and its up projection meet in one lane.
template <int BITS, bool GATED, int NT>
struct WoTiles {
    const int8_t *wb[NT];    // uniform: the tile's channel block, and a lane's place in a chunk of it
    const _Float16 *sb[NT];
    uint32_t wl, sl;
    __device__ __forceinline__ void init(const WoWeight &w0, const WoWeight &w1, int cb0, int lane, int nk32, int G) {
        wl = BITS == 4 ? (lane & 31) * 16 + 8 * (lane >> 5) : lane * 16;
        sl = lane & 31;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const WoWeight &x = GATED && (t & 1) ? w1 : w0;
            const int c = cb0 + (GATED ? t >> 1 : t);
            wb[t] = x.q + (BITS == 4 ? (int64_t)(c >> 1) * nk32 * 1024 + (c & 1) * 512 : (int64_t)c * nk32 * 1024);
            sb[t] = static_cast<const _Float16 *>(x.s) + (BITS == 4 ? (int64_t)(c >> 1) * G * 64 + (c & 1) * 32 : 0);
        }
    }
    // chunk kc's codes and group scales
    __device__ __forceinline__ void load(int kc, const FastDiv &cpg, int G, uint32_t (&w)[NT][BITS / 2], _Float16 (&sc)[NT]) const {
        const int g = BITS == 4 ? min((int)cpg.div(kc), G - 1) : 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if constexpr (BITS == 4) {
                const uint2 v = *reinterpret_cast<const uint2 *>(wb[t] + (int64_t)kc * 1024 + wl);
                w[t][0] = v.x, w[t][1] = v.y;
                sc[t] = (sb[t] + (int64_t)g * 64)[sl];
            } else {
                const uint4 v = *reinterpret_cast<const uint4 *>(wb[t] + (int64_t)kc * 1024 + wl);
                w[t][0] = v.x, w[t][1] = v.y, w[t][2] = v.z, w[t][3] = v.w;
            }
        }
    }
    static __device__ __forceinline__ void widen(const uint32_t (&w)[BITS / 2], int j, f16x2 (&h)[4]) {
        if constexpr (BITS == 4) widen8_q4(w[j], h);
        else widen8_q8(w[2 * j], w[2 * j + 1], h);
    }
};

// acc (scaled like the parts) += the products of the marked blocks first, first + step, ... on the f32
// MFMA, the activations read again.
template <int BITS, bool GATED, int TM, int NT>
__device__ __forceinline__ void wo_marked(const WoRows &p, const WoTiles<BITS, GATED, NT> &tiles, int rb, int first, int step,
                                          f32x16 (&acc)[TM][NT]) {
    const int lane = threadIdx.x & 63, r = lane & 31, nb = p.nkc >> 2, nk32 = p.Kp >> 5;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int row = min(32 * (rb + i) + r, p.M - 1);
        const float up = p.a.scale[row].x;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(up < 0.0f) == 0, 1)) continue;
        const float *a = p.A + (int64_t)row * p.lda;
        for (int b = first; b < nb; b += step) {
            const float s = p.a.mark[((int64_t)(row >> 5) * nb + b) * 32 + (row & 31)] ? -up : 0.0f;
            if (__builtin_amdgcn_ballot_w64(s != 0.0f) == 0) continue;
            for (int kc = 4 * b; kc < min(4 * b + 4, nk32); ++kc) {
                uint32_t w[NT][BITS / 2];
                _Float16 sc[NT];
                tiles.load(kc, p.cpg, p.G, w, sc);
                const int k0 = 32 * kc + 16 * (lane >> 5);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    f32x16 part;
#pragma unroll
                    for (int e = 0; e < 16; ++e) part[e] = 0.0f;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        f16x2 h[4];
                        WoTiles<BITS, GATED, NT>::widen(w[t], j, h);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int k = k0 + 8 * j + e;
                            const float x = a[min(k, p.K - 1)];
                            part = __builtin_amdgcn_mfma_f32_32x32x2f32(k < p.K && s != 0.0f ? x * s : 0.0f,
                                                                        (float)h[e >> 1][e & 1], part, 0, 0, 0);
                        }
                    }
                    const float g = BITS == 4 ? (float)sc[t] : 1.0f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][t][e] = __builtin_fmaf(part[e], g, acc[i][t][e]);
                }
            }
        }
    }
}

// The products of one chunk; read(i, x, j): row block i's part x, step j.
template <int BITS, bool GATED, int TM, int NT, typename Read>
__device__ __forceinline__ void wo_chunk(Read read, const uint32_t (&w)[NT][BITS / 2], const _Float16 (&sc)[NT],
                                         f32x16 (&acc)[TM][NT]) {
    f32x16 part[TM][NT];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        f16x8 p[TM][2], q[NT], ql[NT];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int x = 0; x < 2; ++x) p[i][x] = read(i, x, j);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            f16x2 h[4];
            WoTiles<BITS, GATED, NT>::widen(w[t], j, h);
            q[t] = f16x8{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
            ql[t] = lo_codes(q[t]);
        }
#pragma unroll
        for (int x = 1; x >= 0; --x)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const f16x8 &c = x ? ql[t] : q[t];
                    if (BITS == 8) {
                        acc[i][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[i][x], c, acc[i][t], 0, 0, 0);
                    } else {
                        if (j == 0 && x == 1) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) part[i][t][e] = 0.0f;
                        }
                        part[i][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[i][x], c, part[i][t], 0, 0, 0);
                    }
                }
    }
    if (BITS == 4) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float s = (float)sc[t];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][t][e] = __builtin_fmaf(part[i][t][e], s, acc[i][t][e]);
        }
    }
}

// Stores registers e0 .. e0 + ER - 1 (held in places 0 .. ER - 1) of the tiles at row block rb, channel
// block cb0.
template <int BITS, bool GATED, int TM, int NT, int ER>
__device__ __forceinline__ void wo_store(const WoRows &p, const WoWeight &w0, const WoWeight &w1, const float *b0,
                                         const float *b1, int act, float *C, int64_t ldc, int rb, int cb0, int e0,
                                         const f32x16 (&acc)[TM][NT]) {
    const int lane = threadIdx.x & 63, r = lane & 31;
    float down[TM][ER];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int e = 0; e < ER; ++e) down[i][e] = p.a.scale[min(32 * (rb + i) + acc_row(e0 + e, lane), p.M - 1)].y;
#pragma unroll
    for (int u = 0; u < (GATED ? NT / 2 : NT); ++u) {
        const int n = 32 * (cb0 + u) + r, nn = min(n, p.N - 1);
        const float s0 = BITS == 8 ? static_cast<const float *>(w0.s)[nn] : 1.0f;
        const float s1 = GATED && BITS == 8 ? static_cast<const float *>(w1.s)[nn] : 1.0f;
        const float bg = GATED && b0 ? b0[nn] : kNoBias, bu = GATED && b1 ? b1[nn] : kNoBias;
        if (n >= p.N) continue;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e = 0; e < ER; ++e) {
                const int m = 32 * (rb + i) + acc_row(e0 + e, lane);
                float v = acc[i][GATED ? 2 * u : u][e] * down[i][e] * s0;
                if constexpr (GATED) v = gate_f32(act, v + bg, acc[i][2 * u + 1][e] * down[i][e] * s1 + bu);
                if (m < p.M) C[(int64_t)m * ldc + n] = v;
            }
    }
}

// Pieces: a workgroup computes 32 TM rows x NT tiles, its NW wavefronts splitting K in 64-deep stages.
// Parts and codes go straight into registers, PW stages ahead: no LDS and no barrier in the main loop. The
// shares meet in LDS, each wavefront finishing 16 / NW of the accumulator registers. A piece is one CU's work
// (K = 4096: two wavefronts of a SIMD with 16 chunks each of 128 MFMA cycles and about 50 vector instructions, 4.5
// us) between a start and a joining end: MI355X, K = N = 4096, 4 bits 32 rows 11 us (bf16 tiles 32), 128 rows 19;
// gated int8 14 and 27; the same at N = 1024. More stages in flight gain nothing, 16 x 32 pieces on the 16 x 16
// MFMA neither (gated 4 bits 16 rows 17.8 -> 21.3: as many codes to widen for half of the products).
template <int BITS, bool GATED, int TM, int NT, int NW, int PW>
__global__ __launch_bounds__(64 * NW) void gemm_wo_piece(WoRows p, WoWeight w0, WoWeight w1, const float *__restrict__ b0,
                                                         const float *__restrict__ b1, int act, float *__restrict__ C,
                                                         int64_t ldc, int tilesN) {
    constexpr int CB = GATED ? NT / 2 : NT, ER = 16 / NW, SH = ER * TM * NT * 64;
    static_assert(16 % NW == 0 && (!GATED || NT % 2 == 0), "shares; a tile of each weight");
    __shared__ float red[NW][NW - 1][SH];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int logical = xcd_logical_tile(blockIdx.x, gridDim.x);
    const int rb = (logical / tilesN) * TM, cb0 = (logical % tilesN) * CB;
    const int nk32 = p.Kp >> 5, nst = p.nkc >> 1, last_rb = (p.M - 1) >> 5;
    WoTiles<BITS, GATED, NT> tiles;
    tiles.init(w0, w1, cb0, lane, nk32, p.G);
    f16x8 a[PW][2][TM][2][2];
    uint32_t w[PW][2][NT][BITS / 2];
    _Float16 sc[PW][2][NT];
    const char *pa[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) pa[i] = p.a.parts + (int64_t)min(rb + i, last_rb) * p.nkc * 4096;
    auto load = [&](int slot, int s) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        a[slot][c][i][x][j] =
                            *reinterpret_cast<const f16x8 *>(pa[i] + (int64_t)(2 * s + c) * 4096 + x * 2048 + j * 1024 + (uint32_t)(lane * 16));
            tiles.load(min(2 * s + c, nk32 - 1), p.cpg, p.G, w[slot][c], sc[slot][c]);
        }
    };
    f32x16 acc[TM][NT];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][t][e] = 0.0f;
    if (wave < nst) {
        const int final = wave + (nst - 1 - wave) / NW * NW;  // this wavefront's last stage
#pragma unroll
        for (int d = 0; d < PW; ++d) load(d, min(wave + d * NW, final));
        for (int s0 = wave; s0 < nst; s0 += NW * PW) {
#pragma unroll
            for (int d = 0; d < PW; ++d) {
                const int s = s0 + d * NW;
                if (s >= nst) break;  // uniform
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    wo_chunk<BITS, GATED, TM, NT>([&](int i, int x, int j) { return a[d][c][i][x][j]; }, w[d][c], sc[d][c], acc);
                load(d, min(s + PW * NW, final));
            }
        }
    }
    wo_marked<BITS, GATED, TM, NT>(p, tiles, rb, wave, NW, acc);
    // registers [ER s, ER s + ER) are finished by wavefront s
#pragma unroll
    for (int s = 0; s < NW; ++s) {
        if (s == wave) continue;
        float *d = red[s][wave < s ? wave : wave - 1] + lane;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < ER; ++e) d[((i * NT + t) * ER + e) * 64] = acc[i][t][ER * s + e];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < ER; ++e) {
                float o[NW], v = 0.0f;
#pragma unroll
                for (int s = 0; s < NW; ++s) o[s] = acc[i][t][ER * s + e];
#pragma unroll
                for (int s = 0; s < NW; ++s) v = wave == s ? o[s] : v;
#pragma unroll
                for (int s = 0; s < NW - 1; ++s) v += red[wave][s][((i * NT + t) * ER + e) * 64 + lane];
                acc[i][t][e] = v;
            }
    wo_store<BITS, GATED, TM, NT, ER>(p, w0, w1, b0, b1, act, C, ldc, rb, cb0, ER * wave, acc);
}

// Tiles: 32 TM rows x 4 wavefronts of NT tiles side by side, KS such groups of four on alternate pairs of
// chunks. A chunk's parts pass through LDS once for its four wavefronts (double-buffered), its codes go
// straight into registers, PW stages ahead, and are widened one stage ahead. FP: chunks of a 4-bit
// weight that share a scale (its group is a multiple of 32 FP): their sum is added once, scaled.
//
// MI355X, K = N = 4096, us, least to median: 4 bits 512 rows 45, 4096 rows 258 to 294 (275 GFLOP of f16 MFMA
// work, 194 at 1.42 PFLOP/s); gated int8 512 rows 64 to 66, 4096 rows 472 to 543 (387); gated 4 bits 4096 rows 511
// to 566. Bound by the MFMA together with the widening and scaling (8 vector instructions per MFMA at TM 1), which a
// SIMD's second wavefront covers in part, and at 512 rows by few tiles a CU: 512 x 4096, K = 1024 14.6 us, 4 of them
// MFMA.
template <int BITS, bool GATED, int TM, int NT, int KS, int PW, int FP>
__global__ __launch_bounds__(256 * KS, 2) void gemm_wo_tile(WoRows p, WoWeight w0, WoWeight w1,
                                                                 const float *__restrict__ b0, const float *__restrict__ b1,
                                                                 int act, float *__restrict__ C, int64_t ldc, int tilesN) {
    constexpr int CB = GATED ? NT / 2 : NT, STAGE = KS * TM * 4096, ER = 16 / KS, SH = ER * TM * NT * 64;
    constexpr int RED = KS > 1 ? 4 * KS * (KS - 1) * SH * 4 : 0, LDS = 2 * STAGE > RED ? 2 * STAGE : RED;
    static_assert((PW == 2 || PW == 4) && (KS == 1 || KS == 2) && PW % FP == 0 && (KS == 1 || FP <= 2),
                  "buffers alternate; a group's chunks lie side by side");
    static_assert(!GATED || NT % 2 == 0, "a tile of each weight");
    __shared__ __attribute__((aligned(1024))) char lds[LDS];
    const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ks = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
    const int logical = xcd_logical_tile(blockIdx.x, gridDim.x);
    const int rb = (logical / tilesN) * TM, cb0 = (logical % tilesN) * 4 * CB + wave * CB;
    const int nk32 = p.Kp >> 5, last = p.nkc - 1, last_rb = (p.M - 1) >> 5, nst = p.nkc / KS;
    WoTiles<BITS, GATED, NT> tiles;
    tiles.init(w0, w1, cb0, lane, nk32, p.G);
    u32x4 ra[PW][TM];  // each wavefront moves one part of every row block: plane wave / 2, step wave % 2
    uint32_t w[PW][NT][BITS / 2];
    _Float16 sc[PW][NT];
    const char *pa[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) pa[i] = p.a.parts + (int64_t)min(rb + i, last_rb) * p.nkc * 4096;
    // two neighbouring chunks a group, in turn; past the last stage: a chunk again, not used
    auto chunk = [&](int st) { return min(KS == 1 ? st : 4 * (st >> 1) + 2 * ks + (st & 1), last); };
    auto load_a = [&](int slot, int st) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
            ra[slot][i] = *reinterpret_cast<const u32x4 *>(pa[i] + (int64_t)chunk(st) * 4096 + (uint32_t)(tid * 16));
    };
    auto load_w = [&](int slot, int st) { tiles.load(min(chunk(st), nk32 - 1), p.cpg, p.G, w[slot], sc[slot]); };
    auto store_a = [&](int slot, char *st) {
#pragma unroll
        for (int i = 0; i < TM; ++i) *reinterpret_cast<u32x4 *>(st + (ks * TM + i) * 4096 + tid * 16) = ra[slot][i];
    };
    f16x8 q[2][NT][2];  // the widened codes of a chunk and the next
    float s[NT], sn[NT];
    auto widen = [&](int slot, int at) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f16x2 h[4];
                WoTiles<BITS, GATED, NT>::widen(w[slot][t], j, h);
                q[at][t][j] = f16x8{h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
            }
    };
    f32x16 acc[TM][NT], part[TM][NT];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][t][e] = 0.0f;
#pragma unroll
    for (int d = 0; d < PW; ++d) {
        load_a(d, d);
        load_w(d, d);
    }
    store_a(0, lds);
    load_a(0, PW);
    widen(0, 0);
#pragma unroll
    for (int t = 0; t < NT; ++t) sn[t] = BITS == 4 ? (float)sc[0][t] : 1.0f;
    load_w(0, PW);
    lds_barrier();
    for (int c0 = 0; c0 < nst; c0 += PW) {
#pragma unroll
        for (int d = 0; d < PW; ++d) {
            const int c = c0 + d;
            if (KS * PW > 4 && c >= nst) break;  // uniform
            const char *cur = lds + (d & 1) * STAGE + ks * TM * 4096 + lane * 16;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                f16x8 a[TM][2];
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int x = 0; x < 2; ++x) a[i][x] = *reinterpret_cast<const f16x8 *>(cur + i * 4096 + x * 2048 + j * 1024);
                f16x8 ql[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) ql[t] = lo_codes(q[d & 1][t][j]);
#pragma unroll
                for (int x = 1; x >= 0; --x)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            f32x16 &y = BITS == 4 ? part[i][t] : acc[i][t];
                            if (BITS == 4 && d % FP == 0 && j == 0 && x == 1) {
#pragma unroll
                                for (int e = 0; e < 16; ++e) y[e] = 0.0f;
                            }
                            y = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][x], x ? ql[t] : q[d & 1][t][j], y, 0, 0, 0);
                        }
            }
            // while they run: the next chunk's codes
            widen((d + 1) % PW, (d & 1) ^ 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) s[t] = sn[t], sn[t] = BITS == 4 ? (float)sc[(d + 1) % PW][t] : 1.0f;
            store_a((d + 1) % PW, lds + ((d & 1) ^ 1) * STAGE);
            load_a((d + 1) % PW, c + 1 + PW);
            load_w((d + 1) % PW, c + 1 + PW);
            if (BITS == 4 && d % FP == FP - 1) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][t][e] = __builtin_fmaf(part[i][t][e], s[t], acc[i][t][e]);
            }
            lds_barrier();
        }
    }
    wo_marked<BITS, GATED, TM, NT>(p, tiles, rb, ks, KS, acc);
    if constexpr (KS > 1) {
        // registers [ER g, ER g + ER) are finished by group g
        float *red = reinterpret_cast<float *>(lds);
#pragma unroll
        for (int g = 0; g < KS; ++g) {
            if (g == ks) continue;
            float *d = red + ((g * 4 + wave) * (KS - 1) + (ks < g ? ks : ks - 1)) * SH + lane;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < ER; ++e) d[((i * NT + t) * ER + e) * 64] = acc[i][t][ER * g + e];
        }
        lds_barrier();
        const float *d = red + (ks * 4 + wave) * (KS - 1) * SH + lane;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < ER; ++e) {
                    float v = acc[i][t][e];
#pragma unroll
                    for (int g = 1; g < KS; ++g) v = ks == g ? acc[i][t][ER * g + e] : v;
#pragma unroll
                    for (int g = 0; g < KS - 1; ++g) v += d[g * SH + ((i * NT + t) * ER + e) * 64];
                    acc[i][t][e] = v;
                }
    }
    wo_store<BITS, GATED, TM, NT, ER>(p, w0, w1, b0, b1, act, C, ldc, rb, cb0, ER * ks, acc);
}

}  // namespace enchip
