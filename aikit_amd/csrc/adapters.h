// adapters.h -- low-rank adapters of many requests at once: y_m += B_s (A_s a_m) with s = ids[m], the row's
// slot of a set of adapters (A_s [rank][K], B_s [N][rank], the adapter's scale in B_s). A row whose id is no
// slot gets nothing.
//
// Both products run on the bf16 MFMA with every operand split into three bf16 parts, x = h + m + l, and six
// products of parts summed in f32, as gemm_f32.h does and explains; the set keeps its parts, laid out as the
// MFMA takes them, so that a wavefront loads 64 x 16 contiguous bytes. An operand from 2^-110 up to 2^127 is
// held exactly.
//   adapter_down  t = A_s a for 16 rows by a workgroup, K split over its wavefronts (v_mfma_f32_16x16x32_bf16);
//                 t goes to scratch in parts, laid out for the second product
//   adapter_up    y += B_s t for 32 x 32 outputs by a wavefront (v_mfma_f32_32x32x16_bf16)
// Rows of a block that have different adapters: each adapter among them in turn, from the lowest such row on.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attention_f32.h"
#include "gelu_f32.h"
#include "gemm_f32.h"
#include "kernels.h"

#pragma clang fp contract(off)

namespace enchip {

// A set of adapters and the rows' choice. a: [slot][Kp / 32][R / 16][3][64][8] parts, lane l of a block holding
// rank l % 16 and k 8 (l / 16) ..; b: [slot][Np / 32][R / 16][3][64][8], lane l column l % 32 and rank
// 8 (l / 32) ..; t: [rows / 32][R / 16][3][64][8], lane l row l % 32 and rank 8 (l / 32) ...
struct Adapters {
    const bf16x8 *a, *b;
    bf16x8 *t;
    const int32_t *ids;
    int slots, kb, nb, rt;  // Kp / 32, Np / 32, R / 16
};

__device__ __forceinline__ void split3_8(const float *x, bf16x8 (&p)[3]) {
    float big = 0.0f;
    u32x4 w[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h, m, l;
        split3_pair(x[2 * i], x[2 * i + 1], h, m, l, big);
        w[0][i] = h, w[1][i] = m, w[2][i] = l;
    }
#pragma unroll
    for (int u = 0; u < 3; ++u) p[u] = __builtin_bit_cast(bf16x8, w[u]);
}

// The row's slot, -1 where it has none.
__device__ __forceinline__ int adapter_of(const Adapters &p, int64_t row, int64_t M) {
    const int id = row < M ? p.ids[row] : -1;
    return id >= 0 && id < p.slots ? id : -1;
}

constexpr int AD_ROWS = 16, AD_WAVES = 4;

// VEC: 16-byte loads of a's rows (lda a multiple of 4, a 16-byte aligned, K a multiple of 4).
template <bool VEC>
__global__ __launch_bounds__(64 * AD_WAVES) void adapter_down(const float *__restrict__ a, int64_t lda, int64_t M, int K, Adapters p) {
    __shared__ float red[AD_WAVES][AD_ROWS * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row0 = (int64_t)blockIdx.x * AD_ROWS;
    const int mine = adapter_of(p, row0 + (lane & 15), M);
    const float *src = a + min(row0 + (lane & 15), M - 1) * lda;
    uint32_t todo = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && mine >= 0);
    while (todo != 0) {  // uniform over the workgroup
        const int slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
        const uint32_t rows = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && mine == slot);
        todo &= ~rows;
        for (int rt = 0; rt < p.rt; ++rt) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int kb = wave; kb < p.kb; kb += AD_WAVES) {
                const int k = 32 * kb + 8 * (lane >> 4);
                float x[8];
                if (VEC && k + 8 <= K) {
                    load8(src + k, x);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = k + i < K ? src[k + i] : 0.0f;
                }
                bf16x8 xp[3], ap[3];
                split3_8(x, xp);
                const bf16x8 *at = p.a + ((((int64_t)slot * p.kb + kb) * p.rt + rt) * 3) * 64 + lane;
#pragma unroll
                for (int u = 0; u < 3; ++u) ap[u] = at[64 * u];
                constexpr int pi[6] = {2, 0, 1, 1, 0, 0}, qi[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
                for (int u = 0; u < 6; ++u) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xp[pi[u]], ap[qi[u]], acc, 0, 0, 0);
            }
            // register i of lane l: row 4 (l / 16) + i, rank l % 16
#pragma unroll
            for (int i = 0; i < 4; ++i) red[wave][(4 * (lane >> 4) + i) * 16 + (lane & 15)] = acc[i];
            __syncthreads();
            const int row = tid >> 4, rank = tid & 15;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < AD_WAVES; ++w) v += red[w][tid];
            if ((rows >> row) & 1) {
                float big = 0.0f;
                uint32_t q[3];
                split3_pair(v, 0.0f, q[0], q[1], q[2], big);
                const int64_t m = row0 + row;
                uint16_t *to = reinterpret_cast<uint16_t *>(p.t + ((m >> 5) * p.rt + rt) * 3 * 64 + (m & 31) + 32 * (rank >> 3)) + (rank & 7);
#pragma unroll
                for (int u = 0; u < 3; ++u) to[u * 64 * 8] = (uint16_t)q[u];
            }
            __syncthreads();
        }
    }
}

// The 32 x 32 sums of B_s t at row block mb, column block nb, in the MFMA's accumulator order.
__device__ __forceinline__ f32x16 adapter_tile(const Adapters &p, int mine, int64_t mb, int64_t nb, int lane) {
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
    uint32_t todo = (uint32_t)__builtin_amdgcn_ballot_w64(mine >= 0);
    while (todo != 0) {
        const int slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
        todo &= ~(uint32_t)__builtin_amdgcn_ballot_w64(mine == slot);
        const u32x4 keep = (u32x4)(mine == slot ? ~0u : 0u);
        for (int rt = 0; rt < p.rt; ++rt) {
            const bf16x8 *tp = p.t + (mb * p.rt + rt) * 3 * 64 + lane;
            const bf16x8 *bp = p.b + (((int64_t)slot * p.nb + nb) * p.rt + rt) * 3 * 64 + lane;
            bf16x8 t[1][3], b[1][3];
#pragma unroll
            for (int u = 0; u < 3; ++u) {
                t[0][u] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, tp[64 * u]) & keep);
                b[0][u] = bp[64 * u];
            }
            f32x16 one[1][1] = {{acc}};
            mfma_parts<1, 1>(t, b, one);
            acc = one[0][0];
        }
    }
    return acc;
}

// dst = act(y + B_s t): a wavefront per 32 x 32 outputs, four side by side. dst may be y.
template <bool GELU>
__global__ __launch_bounds__(256) void adapter_up(const float *y, int64_t ldy, float *dst, int64_t ldd, int64_t M, int N, Adapters p,
                                                  int panels) {
    const int lane = threadIdx.x & 63, r = lane & 31;
    const int64_t mb = blockIdx.x / panels, nb = (int64_t)(blockIdx.x % panels) * 4 + (threadIdx.x >> 6);
    const int64_t col = nb * 32 + r;
    if (nb * 32 >= N) return;
    const f32x16 d = adapter_tile(p, adapter_of(p, mb * 32 + r, M), mb, nb, lane);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int64_t row = mb * 32 + acc_row(e, lane);
        if (row >= M || col >= N) continue;
        const float v = y[row * ldy + col] + d[e];
        dst[row * ldd + col] = GELU ? gelu_f32(v) : v;
    }
}

}  // namespace enchip
