// gemm_gated.h -- the gated pair of W8A8 linears on one quantization of the activations:
//   out[m, n] = act(yg) * yu,  y_i = f32(acc_i) aS[m] wS_i[n] (+ bias_i[n]),
// acc_i the exact int32 dots with the gate's and the up projection's codes; y_i rounds as the
// linears' epilogue does (kernels.h dequant).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gated.h"
#include "gemm_pieces.h"
#include "kernels.h"

#pragma clang fp contract(off)

namespace enchip {

struct GatePair {
    const int8_t *w[2];      // fragment-major images of the gate and up weights
    const float *s[2];       // their channel scales
    const float *b[2];       // their biases, or null
};

// One workgroup per CM x CN piece, its NW wavefronts splitting K (gemm_pieces.h), on both weights.
// A is fragment-major at pitch Kp, read up to row m0 + CM - 1.
template <int CM, int CN, int NW>
__global__ __launch_bounds__(64 * NW) void gated_w8a8_piece(const int8_t *__restrict__ A, const float *__restrict__ aS,
                                                            GatePair p, int act, float *__restrict__ out, int64_t ldo, int M,
                                                            int N, int Kp, int piecesN) {
    constexpr int TM = CM / 32, TN = CN / 32, P = CN + 8;
    __shared__ int red[2][NW][CM * P];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = xcd_logical_tile(blockIdx.x, gridDim.x), m0 = (l / piecesN) * CM, n0 = (l % piecesN) * CN;
    const int nk32 = Kp >> 5;
    i32x16 acc[2][TM][TN];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][i][j][e] = 0;
    for (int k = wave; k < nk32; k += NW) {
        i32x4 a[TM], w[2][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
            a[i] = *reinterpret_cast<const i32x4 *>(A + ((int64_t)(m0 / 32 + i) * nk32 + k) * 1024 + lane * 16);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                w[t][j] = *reinterpret_cast<const i32x4 *>(p.w[t] + ((int64_t)(n0 / 32 + j) * nk32 + k) * 1024 + lane * 16);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    acc[t][i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], w[t][j], acc[t][i][j], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    red[t][wave][(32 * i + acc_row(e, lane)) * P + 32 * j + (lane & 31)] = acc[t][i][j][e];
    __syncthreads();
    for (int i = tid; i < CM * CN; i += 64 * NW) {
        const int r = i / CN, c = i % CN, m = m0 + r, n = n0 + c;
        if (m >= M || n >= N) continue;
        float y[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            int s = 0;
#pragma unroll
            for (int k = 0; k < NW; ++k) s += red[t][k][r * P + c];
            y[t] = dequant(s, aS[m], p.s[t][n], p.b[t] ? p.b[t][n] : kNoBias);
        }
        out[(int64_t)m * ldo + n] = gate_f32(act, y[0], y[1]);
    }
}

}  // namespace enchip
