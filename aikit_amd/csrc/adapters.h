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
//   gemm_w8a8_pt_adapters, gemm_w8a8_adapters, gemv_w8a8_adapters: the second product in the epilogue of the W8A8
//                 products, whose rows adapter_down quantizes from the registers that it multiplies
// Rows of a block that have different adapters: each adapter among them in turn, from the lowest such row on.
// What is added to a row without one is -0, the number that leaves every sum as it was: +0 makes a -0 of y's a +0.
//
// Bound by memory where rows are many: 32768 x 1024 to 1024, rank 16, rows of 8 adapters, take 97 to 107 us on MI355X, 41 in
// adapter_down (134 MB of rows, 34 of codes: 4.1 TB/s) and 57 in the product (34 MB of codes, 134 of outputs;
// 69 G int8 operations). A pass of its own for the codes, one for the low-rank parts and one for y took 186. 1500 x 1000
// to 1001 with GELU 8 + 11 us, 512 x 1024 beside 4096 outputs at rank 64 4.5 + 7.4: loads' latency, a workgroup a CU
// or less.
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
// rank l % 16 and k 4 (l / 16) .. + 3 and 16 further (so that a wavefront's 16-byte loads of rows cover whole 64
// bytes); b: [slot][Np / 32][R / 16][3][64][8], lane l column l % 32 and rank
// 8 (l / 32) ..; t: [rows / 32][R / 16][3][64][8], lane l row l % 32 and rank 8 (l / 32) ...
struct Adapters {
    static constexpr bool on = true;
    const bf16x8 *a, *b;
    const float *af;  // A as it is, [slot][R][4 ceil(K / 4)]
    bf16x8 *t;
    const int32_t *ids;
    int slots, kb, nb, rt;  // Kp / 32, Np / 32, R / 16

    // The row's slot, -1 where it has none.
    __device__ __forceinline__ int slot(int64_t row, int64_t M) const {
        const int id = row < M ? ids[row] : -1;
        return id >= 0 && id < slots ? id : -1;
    }
    __device__ __forceinline__ const bf16x8 *t_at(int64_t mb, int rs) const { return t + (mb * rt + rs) * 192; }
    __device__ __forceinline__ const bf16x8 *b_at(int slot, int64_t n, int rs) const {
        return b + (((int64_t)slot * nb + n) * rt + rs) * 192;
    }

    // The column blocks' operands of one slot, kept from one row block to the next.
    template <int TN>
    struct Held {
        int s = -1;
        bf16x8 w[TN][3];
    };

    // The sums of B_s t for the 32 rows of block mb (mine: the slot of row lane % 32) and the TN column blocks
    // from n0 on, as the MFMA's accumulators have them. A row without a slot gets -0.
    template <int TN, class F16>
    __device__ __forceinline__ void tiles(int mine, int64_t mb, int64_t n0, int lane, F16 (&acc)[TN], Held<TN> &held) const {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][e] = -0.0f;
        const uint32_t some = (uint32_t)__builtin_amdgcn_ballot_w64(mine >= 0);
        uint32_t todo = some;
        while (todo != 0) {  // uniform: the adapters among the rows, one after the other
            const int s = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
            todo &= ~(uint32_t)__builtin_amdgcn_ballot_w64(mine == s);
            const u32x4 keep = (u32x4)(mine == s ? ~0u : 0u);
            for (int rs = 0; rs < rt; ++rs) {
                const bf16x8 *tp = t_at(mb, rs) + lane;
                bf16x8 x[1][3];
#pragma unroll
                for (int u = 0; u < 3; ++u) x[0][u] = tp[64 * u];
                if (s != held.s || rt > 1) {
#pragma unroll
                    for (int j = 0; j < TN; ++j)
#pragma unroll
                        for (int u = 0; u < 3; ++u) held.w[j][u] = b_at(s, n0 + j, rs)[64 * u + lane];
                    held.s = s;
                }
#pragma unroll
                for (int u = 0; u < 3; ++u) x[0][u] = __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, x[0][u]) & keep);
                f32x16 d[1][TN];
#pragma unroll
                for (int j = 0; j < TN; ++j) d[0][j] = acc[j];
                mfma_parts<1, TN>(x, held.w, d);
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[j] = d[0][j];
            }
        }
        if (some != 0 && some != ~0u) {  // the others' zeros became +0 in the products
            const uint32_t none = ~some >> acc_row(0, lane);
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    acc[j][e] = __uint_as_float(__float_as_uint(acc[j][e]) | ((none << (31 - acc_row(e, 0))) & 0x80000000u));
        }
    }

    // One output's sum in a thread, for few rows: the first 16 ranks' operands are loaded ahead (dot_begin), the
    // rest in dot_end. x = h + m + l holds exactly.
    struct Dot {
        int s;
        bf16x8 x[2][3], w[2][3];
    };
    __device__ __forceinline__ void dot_load(Dot &d, int row, int64_t n, int c, int rs) const {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < 3; ++u) {
                d.x[h][u] = t_at(row >> 5, rs)[64 * u + (row & 31) + 32 * h];
                d.w[h][u] = b_at(d.s, n, rs)[64 * u + c + 32 * h];
            }
    }
    __device__ __forceinline__ void dot_begin(Dot &d, int row, int64_t M, int64_t n, int c) const {
        d.s = slot(row, M);
        if (d.s >= 0) dot_load(d, row, n, c, 0);
    }
    __device__ __forceinline__ float dot_end(Dot &d, int row, int64_t M, int64_t n, int c) const {
        float sum = 0.0f;
        if (d.s < 0) return -0.0f;
        for (int rs = 0; rs < rt; ++rs) {
            if (rs > 0) dot_load(d, row, n, c, rs);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = (float)d.x[h][0][e] + ((float)d.x[h][1][e] + (float)d.x[h][2][e]);
                    const float w = (float)d.w[h][0][e] + ((float)d.w[h][1][e] + (float)d.w[h][2][e]);
                    sum = __builtin_fmaf(x, w, sum);
                }
        }
        return sum;
    }

    // Few rows of few products in one launch (gemv_w8a8_q, kernels.h): every workgroup forms its rows' low-rank parts
    // itself, a row a wavefront, from the f32 A and the row that the wavefront quantizes; they meet its outputs' B
    // in LDS.
    static constexpr int ROW_RANKS = 32;
    struct Row {
        int mine, s;  // the slots of the wavefront's row and of the thread's output
        bf16x8 w[2][3];
    };
    __device__ __forceinline__ static float *row_t() {
        __shared__ float t[GVQ_ROWS][ROW_RANKS];
        return &t[0][0];
    }
    __device__ __forceinline__ void b_load(Row &d, int64_t n, int c, int rs) const {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < 3; ++u) d.w[h][u] = b_at(d.s, n, rs)[64 * u + c + 32 * h];
    }
    __device__ __forceinline__ void row_begin(Row &d, int row0, int wave, int M, int64_t n, int tid) const {
        d.mine = slot(row0 + wave, M);
        d.s = tid < GVQ_ROWS * 32 ? slot(row0 + (tid >> 5), M) : -1;
        if (d.s >= 0) b_load(d, n, tid & 31, 0);
    }
    template <int QCH>
    __device__ __forceinline__ void row_down(const Row &d, const float4 (&v)[QCH], int K4, int wave, int lane) const {
        if (d.mine < 0) return;  // uniform
        const float4 *at = reinterpret_cast<const float4 *>(af) + (int64_t)d.mine * 16 * rt * K4;
        for (int j0 = 0; j0 < 16 * rt; j0 += 8) {
            float4 x[8][QCH];
            float sum[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < QCH; ++c)  // past K v is zero
                    x[j][c] = at[(int64_t)(j0 + j) * K4 + min(lane + 64 * c, K4 - 1)];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum[j] = 0.0f;
#pragma unroll
                for (int c = 0; c < QCH; ++c) {
                    sum[j] = __builtin_fmaf(v[c].x, x[j][c].x, sum[j]);
                    sum[j] = __builtin_fmaf(v[c].y, x[j][c].y, sum[j]);
                    sum[j] = __builtin_fmaf(v[c].z, x[j][c].z, sum[j]);
                    sum[j] = __builtin_fmaf(v[c].w, x[j][c].w, sum[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum[j] += __uint_as_float(lane_dpp<0xB1>(__float_as_uint(sum[j])));
                sum[j] += __uint_as_float(lane_dpp<0x4E>(__float_as_uint(sum[j])));
                sum[j] += __uint_as_float(lane_dpp<0x141>(__float_as_uint(sum[j])));
                sum[j] += __uint_as_float(lane_dpp<0x140>(__float_as_uint(sum[j])));
                uint32_t p, q;
                lane_swap16(__float_as_uint(sum[j]), p, q);
                sum[j] = __uint_as_float(p) + __uint_as_float(q);
                lane_swap32(__float_as_uint(sum[j]), p, q);
                sum[j] = __uint_as_float(p) + __uint_as_float(q);
                if (lane == 0) row_t()[wave * ROW_RANKS + j0 + j] = sum[j];
            }
        }
    }
    __device__ __forceinline__ float row_up(Row &d, int i, int64_t n, int c) const {
        float sum = 0.0f;
        if (d.s < 0) return -0.0f;
        for (int rs = 0; rs < rt; ++rs) {
            if (rs > 0) b_load(d, n, c, rs);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float w = (float)d.w[h][0][e] + ((float)d.w[h][1][e] + (float)d.w[h][2][e]);
                    sum = __builtin_fmaf(row_t()[i * ROW_RANKS + 16 * rs + 8 * h + e], w, sum);
                }
        }
        return sum;
    }
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

// pack_codes_normal's codes (kernels.h): the conversion to whole numbers is itself the truncation, and a byte
// permute joins two codes.
__device__ __forceinline__ int pack4(float4 v, float inv) {
    const float h = __uint_as_float(0x3effffffu);
    const float a = v.x * inv, b = v.y * inv, c = v.z * inv, d = v.w * inv;
    const uint32_t p = (uint32_t)cvt_i32_f32(a + __builtin_copysignf(h, a)), q = (uint32_t)cvt_i32_f32(b + __builtin_copysignf(h, b));
    const uint32_t r = (uint32_t)cvt_i32_f32(c + __builtin_copysignf(h, c)), t = (uint32_t)cvt_i32_f32(d + __builtin_copysignf(h, d));
    return (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(t, r, 0x0c0c0400u), __builtin_amdgcn_perm(q, p, 0x0c0c0400u), 0x05040100u);
}

// Where adapter_down leaves the rows' codes for a W8A8 product: q[M][ldq] row-major or fragment-major
// (kernels.h frag_off), columns [K, ldq) zero, and their scales.
struct RowCodes {
    int8_t *q;
    float *scale;
    int64_t ldq;
    bool frag;
};

// Grid (ceil(M / 16), y): of the set's R / 16 rank tiles a workgroup takes RTM at a time, blockIdx.y first. K is
// split over the NW wavefronts, 32 deep blocks w, w + NW, ...; KBW of a wavefront's are in flight together, and with
// CODES all of them (ldq <= 32 NW KBW), for the rows are quantized from those registers (by the first of the y).
// VEC: 16-byte loads of a's rows (lda and K multiples of 4, a 16-byte aligned). The barriers order LDS alone: loads
// and stores stay in flight.
template <bool VEC, bool CODES, int NW, int KBW, int RTM>
__global__ __launch_bounds__(64 * NW, 4) void adapter_down(const float *__restrict__ a, int64_t lda, int64_t M, int K, Adapters p,
                                                           RowCodes out) {
    __shared__ float red[NW][RTM * 256];
    __shared__ float top[NW][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * 16, row = row0 + (lane & 15);
    const int mine = p.slot(row, M);
    const float *src = a + min(row, M - 1) * lda;
    float x[KBW][8];
    auto load = [&](int c) {  // the wavefront's blocks of chunk c; zeros past K
#pragma unroll
        for (int i = 0; i < KBW; ++i) {
            const int k = 32 * (NW * (c * KBW + i) + wave) + 4 * g;
            if constexpr (VEC) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(src + min(k + 16 * h, K - 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i][4 * h + e] = v[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] = src[min(k + (e & 3) + 4 * (e & 4), K - 1)];
            }
        }
#pragma unroll
        for (int i = 0; i < KBW; ++i) {
            const int k = 32 * (NW * (c * KBW + i) + wave);
            if (k + 32 <= K) continue;  // uniform
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + 4 * g + (e & 3) + 4 * (e & 4) >= K) x[i][e] = 0.0f;
        }
    };
    load(0);
    if (CODES && blockIdx.y == 0) {  // uniform
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < KBW; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = absmax_step(m, x[i][e]);
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        if (lane < 16) top[wave][lane] = m;
        lds_barrier();
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, top[w][lane & 15]);
        const bool zero = m == 0.0f;
        const float s = zero ? 0.0f : m / 127.0f, inv = zero ? 0.0f : 1.0f / s;
        if (row < M) {
            if (wave == 0 && lane < 16) out.scale[row] = s;
#pragma unroll
            for (int i = 0; i < KBW; ++i) {
                const int kb = NW * i + wave, k = 32 * kb + 4 * g;
                if (32 * kb >= out.ldq) continue;
                const float4 lo = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]), hi = make_float4(x[i][4], x[i][5], x[i][6], x[i][7]);
                int2 c = make_int2(0, 0);
                if (s >= 0x1p-126f) c = make_int2(pack4(lo, inv), pack4(hi, inv));
                else if (!zero) c = make_int2(pack_codes(lo, inv), pack_codes(hi, inv));
                int8_t *to = out.q + (out.frag ? frag_off(row, k, out.ldq >> 5) : row * out.ldq + k);
                *reinterpret_cast<int *>(to) = c.x;
                *reinterpret_cast<int *>(to + (out.frag ? 512 : 16)) = c.y;
            }
        }
    }
    uint32_t todo = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && mine >= 0);
    const int chunks = CODES ? 1 : (p.kb + NW * KBW - 1) / (NW * KBW);
    int held = 0;  // the chunk in x
    while (todo != 0) {  // uniform over the workgroup: the adapters among the rows, one after the other
        const int slot = __builtin_amdgcn_readlane(mine, __builtin_ctz(todo));
        const uint32_t rows = (uint32_t)__builtin_amdgcn_ballot_w64(lane < 16 && mine == slot);
        todo &= ~rows;
        for (int rt0 = blockIdx.y * RTM; rt0 < p.rt; rt0 += gridDim.y * RTM) {
            f32x4 acc[RTM];
#pragma unroll
            for (int j = 0; j < RTM; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            for (int c = 0; c < chunks; ++c) {
                if (!CODES && c != held) load(held = c);
#pragma unroll
                for (int i = 0; i < KBW; ++i) {
                    const int kb = NW * (c * KBW + i) + wave;
                    if (kb >= p.kb) break;  // uniform
                    bf16x8 xp[3];
                    split3_8(x[i], xp);
                    const bf16x8 *at = p.a + (((int64_t)slot * p.kb + kb) * p.rt + rt0) * 192 + lane;
#pragma unroll
                    for (int j = 0; j < RTM; ++j) {
                        if (RTM > 1 && rt0 + j >= p.rt) break;
                        constexpr int pi[6] = {2, 0, 1, 1, 0, 0}, qi[6] = {0, 2, 1, 0, 1, 0};
                        bf16x8 ap[3];
#pragma unroll
                        for (int u = 0; u < 3; ++u) ap[u] = at[192 * j + 64 * u];
#pragma unroll
                        for (int u = 0; u < 6; ++u) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xp[pi[u]], ap[qi[u]], acc[j], 0, 0, 0);
                    }
                }
            }
            // register i of lane l: row 4 (l / 16) + i, rank l % 16
#pragma unroll
            for (int j = 0; j < RTM; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) red[wave][256 * j + (4 * g + i) * 16 + (lane & 15)] = acc[j][i];
            lds_barrier();
            for (int o = tid; o < 256 * RTM; o += 64 * NW) {
                const int rt = rt0 + (o >> 8), r = (o >> 4) & 15, rank = o & 15;
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < NW; ++w) v += red[w][o];
                if (((rows >> r) & 1) && rt < p.rt) {
                    float big = 0.0f;
                    uint32_t q[3];
                    split3_pair(v, 0.0f, q[0], q[1], q[2], big);
                    const int64_t m = row0 + r;
                    uint16_t *to = reinterpret_cast<uint16_t *>(p.t + ((m >> 5) * p.rt + rt) * 192 + (m & 31) + 32 * (rank >> 3)) + (rank & 7);
#pragma unroll
                    for (int u = 0; u < 3; ++u) to[u * 512] = (uint16_t)q[u];
                }
            }
            lds_barrier();
        }
    }
}

// dst = y + B_s t: a wavefront per 32 x 32 outputs, four side by side. dst may be y.
[[maybe_unused]] static __global__ __launch_bounds__(256) void adapter_up(const float *y, int64_t ldy, float *dst,
                                                                          int64_t ldd, int64_t M, int N, Adapters p, int panels) {
    const int lane = threadIdx.x & 63, r = lane & 31;
    const int64_t mb = blockIdx.x / panels, nb = (int64_t)(blockIdx.x % panels) * 4 + (threadIdx.x >> 6);
    const int64_t col = nb * 32 + r;
    if (nb * 32 >= N) return;
    const int mine = p.slot(mb * 32 + r, M);
    float was[16];
    const float *from = y + min(col, (int64_t)N - 1);
#pragma unroll
    for (int e = 0; e < 16; ++e) was[e] = from[min(mb * 32 + acc_row(e, lane), M - 1) * ldy];
    f32x16 d[1];
    Adapters::Held<1> held;
    p.tiles<1>(mine, mb, nb, lane, d, held);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int64_t row = mb * 32 + acc_row(e, lane);
        if (row < M && col < N) dst[row * ldd + col] = was[e] + d[0][e];
    }
}

// The W8A8 product of at most 32 rows with their adapters (kernels.h's gemv_w8a8, which see).
template <int EPI, int NB>
__global__ __launch_bounds__(64 * GV_WAVES) void gemv_w8a8_adapters(
    const int8_t *__restrict__ A, int64_t lda, const int8_t *__restrict__ Wf,
    const float *__restrict__ aS, const float *__restrict__ wS, const float *__restrict__ bias,
    void *__restrict__ out, int64_t ldo, int M, int N, int Kp, Adapters p) {
    gemv_w8a8_body<EPI, NB>(A, lda, Wf, aS, wS, bias, out, ldo, M, N, Kp, p);
}

// The same in one launch, the rows quantized and their low-rank parts formed by every workgroup (16 rows, K = 384,
// N = 1536, rank 8: 5.8 us, where two launches take 11, and 22 for 16 different adapters).
template <int EPI, int QCH>
__global__ __launch_bounds__(64 * GVQ_WAVES) void gemv_w8a8_q_adapters(
    const float *__restrict__ a, const int8_t *__restrict__ Wf, const float *__restrict__ wS,
    const float *__restrict__ bias, void *__restrict__ out, int64_t ldo, int M, int N, int K, int Kp, Adapters p) {
    gemv_w8a8_q_body<EPI, QCH>(a, Wf, wS, bias, out, ldo, M, N, K, Kp, p);
}

// An adapter's parts from A [R][K] and B [N][R]: blocks of 256 threads, first those of A (32 kb x 16 rt values,
// with zeros past K and R), then those of B (scale B rounded once).
[[maybe_unused]] static __global__ __launch_bounds__(256) void adapter_pack(
    const float *__restrict__ A, const float *__restrict__ B, double scale, int K, int N, int R, int kb, int nb, int rt,
    bf16x8 *__restrict__ pa, bf16x8 *__restrict__ pb, float *__restrict__ fa) {
    const int64_t na = (int64_t)kb * rt * 64, i = (int64_t)blockIdx.x * 256 + threadIdx.x;  // 8 values a thread
    float x[8];
    bf16x8 p[3];
    if (i < na) {
        const int lane = (int)(i & 63), K4 = (K + 3) / 4;
        const int64_t block = i >> 6;
        const int j = 16 * (int)(block % rt) + (lane & 15), k0 = 32 * (int)(block / rt) + 4 * (lane >> 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int k = k0 + (e & 3) + 4 * (e & 4);  // Adapters::a's order
            x[e] = j < R && k < K ? A[(int64_t)j * K + k] : 0.0f;
            if (k < 4 * K4) fa[(int64_t)j * 4 * K4 + k] = x[e];
        }
        split3_8(x, p);
#pragma unroll
        for (int u = 0; u < 3; ++u) pa[(block * 3 + u) * 64 + lane] = p[u];
    } else if (i - na < (int64_t)nb * rt * 64) {
        const int lane = (int)((i - na) & 63);
        const int64_t block = (i - na) >> 6;
        const int j0 = 16 * (int)(block % rt) + 8 * (lane >> 5);
        const int64_t n = 32 * (block / rt) + (lane & 31);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = j0 + e < R && n < N ? (float)(scale * (double)B[n * R + j0 + e]) : 0.0f;
        split3_8(x, p);
#pragma unroll
        for (int u = 0; u < 3; ++u) pb[(block * 3 + u) * 64 + lane] = p[u];
    }
}

}  // namespace enchip
