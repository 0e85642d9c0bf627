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

#include <utility>

#include "gated.h"
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

// v of lane B of each 16-lane row, in every lane of the row.
template <int B>
__device__ __forceinline__ float row_lane(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), 0x150 | B, 0xf, 0xf, true));
}

// A few rows: every wavefront covers 16 channels x 4 units of k (32 k of a 4-bit weight, 16 of an
// int8 one: 16 bytes per lane), its four 16-lane rows one unit each. A lane holds 1/16 of its
// unit's activations, which reach the row's 16 channels as broadcasts within the row. The
// WO_WAVES wavefronts of a workgroup split K; the sums meet in LDS and are added in one order.
// PF: steps whose loads are in flight together.
constexpr int WO_WAVES = 8;

template <int BITS, int MB, bool GATED, int PF>
__global__ __launch_bounds__(64 * WO_WAVES) void gemv_wo(const float *__restrict__ A, int64_t lda, WoWeight w0, WoWeight w1,
                                                         const float *__restrict__ b0, const float *__restrict__ b1, int act,
                                                         float *__restrict__ C, int64_t ldc, int M, int N, int K, int Kp,
                                                         int cpg, int G, int tilesN) {
    constexpr int NWT = GATED ? 2 : 1, CK = BITS == 4 ? 32 : 16, AV = CK / 16;
    __shared__ float red[NWT][MB][WO_WAVES][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, part = lane >> 4, i = lane & 15;
    const int n0 = (blockIdx.x % tilesN) * 16, m0 = (blockIdx.x / tilesN) * MB;
    const int units = Kp / CK;
    const WoWeight w[2] = {w0, w1};
    const float *ar[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) ar[m] = A + (int64_t)min(m0 + m, M - 1) * lda;

    float sum[NWT][MB];
#pragma unroll
    for (int t = 0; t < NWT; ++t)
#pragma unroll
        for (int m = 0; m < MB; ++m) sum[t][m] = 0.0f;

    for (int s0 = 4 * wave; s0 < units; s0 += 4 * WO_WAVES * PF) {
        uint4 q[PF][NWT];
        float sc[PF][NWT], a[PF][MB][AV];
#pragma unroll
        for (int p = 0; p < PF; ++p) {
            const int u = s0 + 4 * WO_WAVES * p + part, uc = min(u, units - 1);
            const int64_t at = BITS == 4 ? ((int64_t)(n0 >> 6) * (Kp >> 5) + uc) * 1024 + ((n0 & 63) + i) * 16
                                         : ((int64_t)(n0 >> 5) * (Kp >> 5) + (uc >> 1)) * 1024 + ((n0 & 31) + i + 32 * (uc & 1)) * 16;
#pragma unroll
            for (int t = 0; t < NWT; ++t) {
                q[p][t] = *reinterpret_cast<const uint4 *>(w[t].q + at);
                if (BITS == 4)
                    sc[p][t] = (float)static_cast<const _Float16 *>(
                        w[t].s)[((int64_t)(n0 >> 6) * G + min(uc / cpg, G - 1)) * 64 + (n0 & 63) + i];
            }
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int e = 0; e < AV; ++e) {
                    const int k = CK * u + AV * i + e;
                    const float v = ar[m][min(k, K - 1)];
                    a[p][m][e] = k < K ? v : 0.0f;
                }
        }
#pragma unroll
        for (int p = 0; p < PF; ++p)
#pragma unroll
            for (int t = 0; t < NWT; ++t) {
                float g[MB];  // the unit's sums, unscaled
#pragma unroll
                for (int m = 0; m < MB; ++m) g[m] = 0.0f;
                const uint32_t qd[4] = {q[p][t].x, q[p][t].y, q[p][t].z, q[p][t].w};
                auto dword = [&](auto dc) {
                    constexpr int D = decltype(dc)::value;
                    const uint32_t lo = qd[D];
                    uint32_t hi = lo >> 4;
                    if (BITS == 4) asm("" : "+v"(hi));  // one shift for its four codes
                    auto byte = [&](auto bc) {
                        constexpr int B = decltype(bc)::value, J = 4 * D + B;
                        if constexpr (BITS == 4) {
                            const float f0 = __builtin_amdgcn_cvt_off_f32_i4((int)((lo >> (8 * B)) & 0xff));  // q / 16
                            const float f1 = __builtin_amdgcn_cvt_off_f32_i4((int)((hi >> (8 * B)) & 0xff));
#pragma unroll
                            for (int m = 0; m < MB; ++m) {
                                g[m] = __builtin_fmaf(row_lane<J>(a[p][m][0]), f0, g[m]);
                                g[m] = __builtin_fmaf(row_lane<J>(a[p][m][AV - 1]), f1, g[m]);
                            }
                        } else {
                            const float f = (float)(int8_t)((lo >> (8 * B)) & 0xff);
#pragma unroll
                            for (int m = 0; m < MB; ++m) g[m] = __builtin_fmaf(row_lane<J>(a[p][m][0]), f, g[m]);
                        }
                    };
                    [&]<int... B>(std::integer_sequence<int, B...>) { (byte(std::integral_constant<int, B>{}), ...); }
                    (std::make_integer_sequence<int, 4>{});
                };
                [&]<int... D>(std::integer_sequence<int, D...>) { (dword(std::integral_constant<int, D>{}), ...); }
                (std::make_integer_sequence<int, 4>{});
#pragma unroll
                for (int m = 0; m < MB; ++m)
                    sum[t][m] = BITS == 4 ? __builtin_fmaf(g[m], 16.0f * sc[p][t], sum[t][m]) : sum[t][m] + g[m];
            }
    }
#pragma unroll
    for (int t = 0; t < NWT; ++t)
#pragma unroll
        for (int m = 0; m < MB; ++m) red[t][m][wave][lane] = sum[t][m];
    __syncthreads();
    if (tid >= 16 * MB) return;
    const int m = tid >> 4, n = n0 + i;
    if (m0 + m >= M || n >= N) return;
    float y[NWT];
#pragma unroll
    for (int t = 0; t < NWT; ++t) {
        y[t] = 0.0f;
#pragma unroll
        for (int j = 0; j < WO_WAVES; ++j)
#pragma unroll
            for (int p = 0; p < 4; ++p) y[t] += red[t][m][j][16 * p + i];
        if (BITS == 8) y[t] *= static_cast<const float *>(w[t].s)[n];
    }
    float v = y[0];
    if constexpr (GATED) v = gate_f32(act, b0 ? y[0] + b0[n] : y[0], b1 ? y[1] + b1[n] : y[1]);
    C[(int64_t)(m0 + m) * ldc + n] = v;
}

}  // namespace enchip
