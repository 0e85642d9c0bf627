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

// act(yg) * yu for four neighbouring outputs of a row.
template <int ACT>
__device__ __forceinline__ f32x4 gate4(const int4 &g, const int4 &u, float as, const float4 (&ws)[2], const float4 (&bb)[2]) {
    auto one = [&](int ag, int au, float sg, float su, float bg, float bu) {
        return gate_f32(ACT, dequant(ag, as, sg, bg), dequant(au, as, su, bu));
    };
    return f32x4{one(g.x, u.x, ws[0].x, ws[1].x, bb[0].x, bb[1].x), one(g.y, u.y, ws[0].y, ws[1].y, bb[0].y, bb[1].y),
                 one(g.z, u.z, ws[0].z, ws[1].z, bb[0].z, bb[1].z), one(g.w, u.w, ws[0].w, ws[1].w, bb[0].w, bb[1].w)};
}

// Up to 32 rows, quantized by the workgroups that use them: gemv_w8a8_q (kernels.h) on both
// weights, one launch. A workgroup quantizes 8 rows into LDS, its 8 wavefronts split K for 32
// output channels of the gate and of the up projection. K % 4 == 0, K <= 256 QCH, 16-byte aligned
// rows; dynamic LDS gated_q_lds_bytes(Kp). Bound by the launch and one trip to memory: MI355X, 16 rows, K =
// 384, N = 1536 3.8 us (quantization and pieces 6.6); K = N = 4096 13.0 (15.5), 33.6 MB.
__host__ __device__ inline int gated_q_lds_bytes(int Kp) { return Kp * 32 + 2 * GVQ_WAVES * GVQ_ROWS * 32 * 4 + 64; }

template <int QCH>
__global__ __launch_bounds__(64 * GVQ_WAVES) void gated_w8a8_q(const float *__restrict__ a, GatePair p, int act,
                                                               float *__restrict__ out, int64_t ldo, int M, int N, int K,
                                                               int Kp) {
    extern __shared__ __attribute__((aligned(16))) int8_t gvq[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nb = blockIdx.x, rg = blockIdx.y, nk32 = Kp >> 5, K4 = K >> 2, Kp4 = Kp >> 2;
    int *red = reinterpret_cast<int *>(gvq + Kp * 32);
    float *s_as = reinterpret_cast<float *>(red + 2 * GVQ_WAVES * GVQ_ROWS * 32);
    const int row = rg * GVQ_ROWS + wave;  // the row this wavefront quantizes
    float4 v[QCH];
    if (row < M) {
        const i32x4 *src = reinterpret_cast<const i32x4 *>(a + (int64_t)row * K);
#pragma unroll
        for (int c = 0; c < QCH; ++c) {
            const int k4 = lane + 64 * c;
            const i32x4 t = src[min(k4, K4 - 1)];
            const int keep = k4 < K4 ? -1 : 0;
            v[c] = make_float4(__int_as_float(t.x & keep), __int_as_float(t.y & keep), __int_as_float(t.z & keep),
                               __int_as_float(t.w & keep));
        }
    }
    // this wavefront's weight fragments wave, wave + 8, ... (clamped; extra copies skipped below)
    i32x4 b[2][QCH];
#pragma unroll
    for (int u = 0; u < QCH; ++u)
#pragma unroll
        for (int t = 0; t < 2; ++t)
            b[t][u] = *reinterpret_cast<const i32x4 *>(
                p.w[t] + ((int64_t)nb * nk32 + min(wave + u * GVQ_WAVES, nk32 - 1)) * 1024 + lane * 16);
    if (row < M) {
        const float m = row_absmax<QCH>(v);
        const bool zero = m == 0.0f;
        const float sc = zero ? 0.0f : m / 127.0f;
        const float inv = zero ? 0.0f : 1.0f / sc;
#pragma unroll
        for (int c = 0; c < QCH; ++c) {
            const int k4 = lane + 64 * c;
            if (k4 < Kp4)
                *reinterpret_cast<int *>(gvq + frag_off(row & 31, 4 * (int64_t)k4, nk32)) =
                    (!zero && k4 < K4) ? pack_codes(v[c], inv) : 0;
        }
        if (lane == 0) s_as[wave] = sc;
    }
    __syncthreads();
    i32x16 acc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0;
#pragma unroll
    for (int u = 0; u < QCH; ++u) {
        const int kk = wave + u * GVQ_WAVES;
        if (kk < nk32) {
            const i32x4 av = *reinterpret_cast<const i32x4 *>(gvq + kk * 1024 + lane * 16);
#pragma unroll
            for (int t = 0; t < 2; ++t) acc[t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av, b[t][u], acc[t], 0, 0, 0);
        }
    }
    // the group's rows 8q .. 8q + 7 of the 32-row tile are registers 4q .. 4q + 3
    const int q = rg & 3;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            red[((t * GVQ_WAVES + wave) * GVQ_ROWS + (lane >> 5) * 4 + i) * 32 + (lane & 31)] = acc[t][4 * q + i];
    __syncthreads();
    if (tid >= GVQ_ROWS * 32) return;
    const int i = tid >> 5, c = tid & 31, orow = rg * GVQ_ROWS + i, col = nb * 32 + c;
    if (orow >= M || col >= N) return;
    float y[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        int sum = 0;
#pragma unroll
        for (int w = 0; w < GVQ_WAVES; ++w) sum += red[((t * GVQ_WAVES + w) * GVQ_ROWS + i) * 32 + c];
        y[t] = dequant(sum, s_as[i], p.s[t][col], p.b[t] ? p.b[t][col] : kNoBias);
    }
    out[(int64_t)orow * ldo + col] = gate_f32(act, y[0], y[1]);
}

// One workgroup per CM x CN piece, its 4 wavefronts splitting K in 64-deep stages, two of them in
// flight (gemm_pieces.h), on both weights. Any M, N and alignment. A is fragment-major at pitch Kp,
// read up to row m0 + CM - 1. Bound by what a CU reads for its pieces (2 CN + CM codes per k), its MFMAs
// an eighth of the time: MI355X 1500 x 1001, K = 1000 13 to 14 us, K = N = 4096 256 rows 22.
template <int CM, int CN, int ACT>
__global__ __launch_bounds__(256, 2) void gated_w8a8_piece(const int8_t *__restrict__ A, const float *__restrict__ aS,
                                                           GatePair p, float *__restrict__ out, int64_t ldo, int M, int N,
                                                           int Kp, int piecesN) {
    constexpr int TM = CM / 32, TN = CN / 32, NW = 4, PW = 2, P = CN + 8, RL = CN / 4, NG = CM * RL / 256;
    static_assert(CM * RL % 256 == 0, "whole passes");
    __shared__ __attribute__((aligned(16))) int red[2][NW][CM * P];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l = xcd_logical_tile(blockIdx.x, gridDim.x), m0 = (l / piecesN) * CM, n0 = (l % piecesN) * CN;
    const int nst = Kp / PC_BK, nk32 = Kp >> 5;
    i32x4 a[PW][2][TM], w[PW][2][2][TN];
    auto load = [&](int slot, int s) {  // this wavefront's s-th stage
        const int64_t k32 = 2 * (int64_t)(wave + s * NW);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
                a[slot][kb][i] = *reinterpret_cast<const i32x4 *>(A + ((int64_t)(m0 / 32 + i) * nk32 + k32 + kb) * 1024 + lane * 16);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    w[slot][kb][t][j] =
                        *reinterpret_cast<const i32x4 *>(p.w[t] + ((int64_t)(n0 / 32 + j) * nk32 + k32 + kb) * 1024 + lane * 16);
        }
    };
    i32x16 acc[2][TM][TN];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[t][i][j][e] = 0;
    const int ns = nst > wave ? (nst - wave + NW - 1) / NW : 0;  // uniform
    if (ns > 0) {
#pragma unroll
        for (int d = 0; d < PW; ++d) load(d, min(d, ns - 1));
        for (int s = 0; s < ns; s += PW) {
#pragma unroll
            for (int d = 0; d < PW; ++d) {
                if (s + d >= ns) break;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < TM; ++i)
#pragma unroll
                            for (int j = 0; j < TN; ++j)
                                acc[t][i][j] =
                                    __builtin_amdgcn_mfma_i32_32x32x32_i8(a[d][kb][i], w[d][kb][t][j], acc[t][i][j], 0, 0, 0);
                load(d, min(s + PW + d, ns - 1));
            }
        }
    }
    // this thread's outputs: group tid % RL of rows tid / RL + i * 256 / RL
    const int c4 = 4 * (tid % RL), r0 = tid / RL, col = n0 + c4;
    float as[NG];
    float4 ws[2], bb[2];
#pragma unroll
    for (int i = 0; i < NG; ++i) as[i] = aS[min(m0 + r0 + i * (256 / RL), M - 1)];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        auto at = [&](const float *v, int u) { return v[min(col + u, N - 1)]; };
        ws[t] = make_float4(at(p.s[t], 0), at(p.s[t], 1), at(p.s[t], 2), at(p.s[t], 3));
        bb[t] = p.b[t] ? make_float4(at(p.b[t], 0), at(p.b[t], 1), at(p.b[t], 2), at(p.b[t], 3))
                       : make_float4(kNoBias, kNoBias, kNoBias, kNoBias);
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
    const bool vec = N % 4 == 0 && ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int r = r0 + i * (256 / RL), row = m0 + r;
        int4 v[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            v[t] = *reinterpret_cast<const int4 *>(&red[t][0][r * P + c4]);
#pragma unroll
            for (int k = 1; k < NW; ++k) {
                const int4 o = *reinterpret_cast<const int4 *>(&red[t][k][r * P + c4]);
                v[t].x += o.x, v[t].y += o.y, v[t].z += o.z, v[t].w += o.w;
            }
        }
        const f32x4 y = gate4<ACT>(v[0], v[1], as[i], ws, bb);
        if (row >= M) continue;
        float *o = out + (int64_t)row * ldo + col;
        if (vec) {
            if (col < N) *reinterpret_cast<f32x4 *>(o) = y;
        } else {
            const float t[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (col + u < N) o[u] = t[u];
        }
    }
}

// Many rows: gemm_w8a8_pt's main loop (gemm_persistent.h) with a wavefront's two 32-channel blocks
// taken one from each weight, so a workgroup's tile is BM rows x 128 output channels and an output's
// two accumulators meet in the wavefront that holds both. MI355X, 32768 rows, K = 1024, N = 4096, SiLU: 320 us
// the least and 372 to 409 the median of 24 launches (the clock gives way under it), the products
// (0.55 POP) and the writing of 537 MB one after the other: 1024 more of K add 235 us, and
// without its stores it takes 100 less. K = N = 4096, 4096 rows 129 us the least (2.1 POP/s), 136 to 146 the median. Where
// it took 337 us, row segments of 512 bytes through LDS took 349, plain stores, 64-row tiles three a CU and
// panels of 4 or 16 columns 354 to 361; panels of 8 in place of none took medians from 437 to 411. Preconditions as
// there (an even number of 64-deep stages, 32-bit offsets, N % 4 == 0, 16-byte aligned rows of out,
// fragment-major A).
constexpr int GP_BN = 128;  // output channels of a tile
constexpr int GP_PANEL = 8;  // tile columns of a panel

template <int BM, int ACT, int PRIO>
__global__ __launch_bounds__(256, BM == PT_BM_SMALL ? 3 : 2) void gated_w8a8_pt(const int8_t *__restrict__ A,
                                                                                const float *__restrict__ aS, GatePair p,
                                                                                float *__restrict__ out, int64_t ldo, int M,
                                                                                int N, int Kp, int tilesN, int numTiles) {
    constexpr int BK = PT_BK, PW = PT_PW, NW = 4, TM = BM / 32, KB = BK / 32, FA = TM * KB, FAW = FA / NW, STAGE = FA * 1024;
    constexpr int RING_LOADS = FAW + KB * 2, SP = 72;
    static_assert(FA % NW == 0 && PW == 2, "A fragments per stage split over the waves");
    __shared__ __attribute__((aligned(1024))) int8_t smem[2 * STAGE];
    __shared__ __attribute__((aligned(16))) int s_tr[NW][32 * SP];
    __shared__ __attribute__((aligned(16))) float s_as[BM];
    __shared__ __attribute__((aligned(16))) float s_ws[2][GP_BN], s_b[2][GP_BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nk = Kp / BK, nk32 = Kp >> 5;
    // Block b runs on XCD b % 8; each XCD walks a contiguous range of tiles.
    const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, per_xcd = gridDim.x >> 3;
    const int q = numTiles >> 3, r = numTiles & 7;
    const int xbeg = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
    const int xcnt = q + (xcd < r ? 1 : 0);
    const int ntiles = slot < xcnt ? (xcnt - slot + per_xcd - 1) / per_xcd : 0;
    if (ntiles == 0) return;
    // Tiles are numbered panel by panel of GP_PANEL tile columns, row blocks first: what an XCD holds
    // at once is a few row blocks times one panel, whose weights stay in its L2.
    const int rbs = numTiles / tilesN;
    auto tile_at = [&](int i, int &m0, int &n0) {
        const int t = xbeg + slot + i * per_xcd, panel = t / (rbs * GP_PANEL), rest = t - panel * rbs * GP_PANEL;
        const int width = min(GP_PANEL, tilesN - panel * GP_PANEL), rb = rest / width;
        m0 = rb * BM;
        n0 = (panel * GP_PANEL + rest - rb * width) * GP_BN;
    };
    uint32_t aoff_c[FAW], aoff_x[FAW], woff_c, woff_x;  // this lane's offsets: current / next tile
    auto tile_offs = [&](int tile, uint32_t *aoff, uint32_t &woff) {
        int m0, n0;
        tile_at(tile, m0, n0);
#pragma unroll
        for (int i = 0; i < FAW; ++i) {
            const int f = wave + NW * i;
            aoff[i] = (uint32_t)((m0 / 32 + f / KB) * nk32 + f % KB) * 1024u + lane * 16;
        }
        woff = (uint32_t)(n0 / 32 + wave) * (uint32_t)nk32 * 1024u + lane * 16;
    };
    i32x4 wreg[PW][KB][2], areg[PW][FAW];
    auto load_stage = [&](int ring, int ls) {
        const bool nx = ls >= nk;
        const uint32_t t = nx ? ls - nk : ls, wo = nx ? woff_x : woff_c;
#pragma unroll
        for (int i = 0; i < FAW; ++i)
            areg[ring][i] = *reinterpret_cast<const i32x4 *>(A + ((nx ? aoff_x[i] : aoff_c[i]) + t * (KB * 1024)));
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int j = 0; j < 2; ++j) wreg[ring][kb][j] = *reinterpret_cast<const i32x4 *>(p.w[j] + (wo + (t * KB + kb) * 1024u));
    };
    auto awrite = [&](int ls, int ring) {
#pragma unroll
        for (int i = 0; i < FAW; ++i)
            *reinterpret_cast<i32x4 *>(smem + ls * STAGE + (wave + NW * i) * 1024 + lane * 16) = areg[ring][i];
    };
    i32x16 acc[TM][2];
    tile_offs(0, aoff_c, woff_c);
    tile_offs(ntiles > 1 ? 1 : 0, aoff_x, woff_x);
#pragma unroll
    for (int d = 0; d < PW; ++d) load_stage(d, d);
    awrite(0, 0);
    __syncthreads();

    // A lane's outputs: columns 4 c4 .. of rows rsub + 8 k. Rows 4 apart in a 16-lane group start 32
    // banks apart.
    const int c4 = lane & 7, rsub = (lane >> 4) + 4 * ((lane >> 3) & 1);
    const int as_slot = (tid & ~31) + (tid & 7) * 4 + ((tid & 31) >> 3);  // its 4 rows' scales contiguous
    int g = 0;
    for (int it = 0; it < ntiles; ++it) {
        int m0, n0;
        tile_at(it, m0, n0);
        // the tile's epilogue constants, loaded before its main loop, staged in LDS after it
        const float c_as = aS[min(m0 + (tid & (BM - 1)), M - 1)];
        const int cn = min(n0 + (tid & (GP_BN - 1)), N - 1), ct = tid >> 7;
        const float *bt = ct ? p.b[1] : p.b[0];
        const float c_ws = (ct ? p.s[1] : p.s[0])[cn], c_b = bt ? bt[cn] : kNoBias;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
        for (int t0 = 0; t0 < nk; t0 += PW) {
#pragma unroll
            for (int d = 0; d < PW; ++d) {
                const int t = t0 + d;
                const int8_t *base = smem + ((g + t) & 1) * STAGE + lane * 16;
                if (PRIO) __builtin_amdgcn_s_setprio(PRIO);
                i32x4 af[KB][TM];
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < TM; ++i) af[kb][i] = *reinterpret_cast<const i32x4 *>(base + (i * KB + kb) * 1024);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(af[kb][i], wreg[d][kb][j], acc[i][j], 0, 0, 0);
                awrite((g + t + 1) & 1, (d + 1) % PW);
                load_stage(d, t + PW);
                __builtin_amdgcn_sched_group_barrier(0x100, FA, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x200, FAW, 0);
#pragma unroll
                for (int u = 0; u < RING_LOADS; ++u) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, TM * 2 * KB - 2 - RING_LOADS, 0);
                __syncthreads();
            }
        }
        g += nk;
#pragma unroll
        for (int i = 0; i < FAW; ++i) aoff_c[i] = aoff_x[i];
        woff_c = woff_x;
        tile_offs(it + 2 < ntiles ? it + 2 : ntiles - 1, aoff_x, woff_x);

        if (PRIO) __builtin_amdgcn_s_setprio(0);
        if (tid < BM) s_as[as_slot] = c_as;
        s_ws[ct][tid & (GP_BN - 1)] = c_ws;
        s_b[ct][tid & (GP_BN - 1)] = c_b;
        __syncthreads();
        const int lcol = wave * 32 + 4 * c4, col = n0 + lcol;
        float4 ws[2], bb[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            ws[t] = *reinterpret_cast<const float4 *>(&s_ws[t][lcol]);
            bb[t] = *reinterpret_cast<const float4 *>(&s_b[t][lcol]);
        }
        int *scr = s_tr[wave];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) scr[acc_row(e, lane) * SP + j * 32 + (lane & 31)] = acc[i][j][e];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const float4 as4 = *reinterpret_cast<const float4 *>(&s_as[i * 32 + rsub * 4]);
            const float as[4] = {as4.x, as4.y, as4.z, as4.w};
            int4 vg[4], vu[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                vg[k] = *reinterpret_cast<const int4 *>(&scr[(rsub + 8 * k) * SP + 4 * c4]);
                vu[k] = *reinterpret_cast<const int4 *>(&scr[(rsub + 8 * k) * SP + 32 + 4 * c4]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f32x4 y = gate4<ACT>(vg[k], vu[k], as[k], ws, bb);
                const int row = m0 + i * 32 + rsub + 8 * k;
                if (row < M && col < N)
                    __builtin_nontemporal_store(y, reinterpret_cast<f32x4 *>(out + (int64_t)row * ldo + col));
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }
}

}  // namespace enchip
