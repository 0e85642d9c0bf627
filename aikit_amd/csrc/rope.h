// rope.h -- rotary positions on rows of heads.
//
// Row t at position p, pair j < r/2 of every head (freq f_j, mscale m):
//   (y1, y2) = m (x1 cos(p f_j) - x2 sin(p f_j), x2 cos(p f_j) + x1 sin(p f_j)),
// the pair being elements (j, j + r/2) of the head (half) or (2j, 2j + 1) (interleaved);
// elements r .. head_dim pass through.
//
// The angle is formed in turns and reduced in 64 bits (a far position times a frequency keeps no fraction in
// 32): f_j / 2 pi less whole turns is held in two parts, and the product with p is exact (a multiplication
// and what it rounded off) but for 2^-32 turns at the largest frequencies, 2^40. Sine and cosine of the
// reduced angle in 32 bits: with the products' rounding under 2^-21 m (|x1| + |x2|) at any position, where f_j / 2 pi in
// one part left 2^-51 |p f_j| more. The pairs' angles are those of every head of
// the row, so a workgroup computes them once for its rows into LDS and then streams the rows.
//
// Bound by memory: 8 bytes an element. 64 x 512 tokens of 24 heads of 64 (403 MB) take 79 us on MI355X,
// 5.1 TB/s, as a copy does (5.2); half of each of 32 heads of 64, 20011 rows, interleaved, 62 us. One item
// in flight a thread took 109 us (four: 79), single floats in place of 16 bytes 131 us against 62. Rotated
// parts that 16-byte accesses do not divide take 8 or 4 bytes: 32768 rows of 24 heads of 64, 42 rotated,
// interleaved 79 us (4 bytes: 104), half 95 (100); 20 rotated, half 105 (126).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

#pragma clang fp contract(off)

namespace enchip {

constexpr int ROPE_MAX_PAIRS = 512;  // pairs of a head (head_dim up to 1024)
constexpr int ROPE_CS = 2048;        // angles of a workgroup's rows in LDS
constexpr int ROPE_BATCH = 4;        // items of a thread whose loads are in flight together

template <int V>
__device__ __forceinline__ void rope_load(float *v, const float *p) {
    if constexpr (V == 4) {
        const f32x4 t = *reinterpret_cast<const f32x4 *>(p);
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    } else if constexpr (V == 2) {
        const float2 t = *reinterpret_cast<const float2 *>(p);
        v[0] = t.x, v[1] = t.y;
    } else {
        v[0] = p[0];
    }
}
template <int V>
__device__ __forceinline__ void rope_store(const float *v, float *p) {
    if constexpr (V == 4) *reinterpret_cast<f32x4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
    else if constexpr (V == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    else p[0] = v[0];
}

// A workgroup's TR rows, as items: per head first those of the rotated part (half: V elements of each
// half; interleaved: V elements, V / 2 pairs, or with V = 1 one pair), then, not in place, those of the
// passed-through part, RV elements each. ipr: items per head. Every V-wide (RV-wide) access is aligned to
// its size: the launch chooses them so.
template <bool INTERLEAVED, int V, int RV>
__global__ __launch_bounds__(256) void rope_rows(const float *x, int64_t ldx, float *y, int64_t ldy,
                                                 const double2 *__restrict__ turns, float mscale,
                                                 const int32_t *__restrict__ pos, int64_t pos0, int64_t row0, int L,
                                                 int64_t rows, int TR, FastDiv heads, FastDiv ipr, int hd, int r) {
    __shared__ float2 cs[ROPE_CS];
    constexpr bool INNER = INTERLEAVED && V > 1;   // an item's pairs lie within it
    constexpr int PI = INNER ? V / 2 : V;          // pairs of an item
    constexpr int EI = INTERLEAVED && !INNER ? 2 : V;  // elements from one item to the next
    constexpr int W = V > RV ? V : RV;
    const int64_t first = (int64_t)blockIdx.x * TR;
    const int tr = (int)min((int64_t)TR, rows - first), np = r / 2;
    for (int t = threadIdx.x; t < tr * np; t += 256) {
        const int row = t / np, j = t - row * np;
        const double p = pos ? (double)pos[first + row] : (double)(pos0 + (row0 + first + row) % L);
        const double2 f = turns[j];
        const double a = p * f.x, e = __builtin_fma(p, f.y, __builtin_fma(p, f.x, -a));
        float s, c;
        sincospif(2.0f * (float)(a - rint(a) + e), &s, &c);
        cs[t] = make_float2(c * mscale, s * mscale);
    }
    __syncthreads();
    const int rot = np / PI;                       // rotated items of a head
    const int mate = INTERLEAVED ? 1 : np;         // from a pair's first element to its second
    const uint32_t items = (uint32_t)tr * heads.d * ipr.d;
    for (uint32_t i0 = threadIdx.x; i0 < items; i0 += 256 * ROPE_BATCH) {
        float a[ROPE_BATCH][W], b[ROPE_BATCH][V];
        float *dst[ROPE_BATCH];
        int at[ROPE_BATCH];  // the item's first angle, -1: passed through, -2: none
#pragma unroll
        for (int u = 0; u < ROPE_BATCH; ++u) {
            const uint32_t i = i0 + 256 * u;
            if (i >= items) {
                at[u] = -2;
                continue;
            }
            const uint32_t hr = ipr.div(i), row = heads.div(hr);
            const int e = (int)(i - hr * ipr.d), h = (int)(hr - row * heads.d);
            const bool turn = e < rot;
            const int off = h * hd + (turn ? EI * e : r + RV * (e - rot));
            const float *src = x + (first + row) * ldx + off;
            dst[u] = y + (first + row) * ldy + off;
            at[u] = turn ? (int)row * np + PI * e : -1;
            if (V == RV || turn) rope_load<V>(a[u], src);
            else rope_load<RV>(a[u], src);
            if (!INNER && turn) rope_load<V>(b[u], src + mate);
        }
#pragma unroll
        for (int u = 0; u < ROPE_BATCH; ++u) {
            if (at[u] == -2) continue;
            if (at[u] >= 0) {
#pragma unroll
                for (int k = 0; k < PI; ++k) {
                    const float2 w = cs[at[u] + k];
                    float &e1 = INNER ? a[u][2 * k] : a[u][k], &e2 = INNER ? a[u][2 * k + 1] : b[u][k];
                    const float x1 = e1, x2 = e2;
                    e1 = x1 * w.x - x2 * w.y;
                    e2 = x2 * w.x + x1 * w.y;
                }
                if constexpr (!INNER) rope_store<V>(b[u], dst[u] + mate);
            }
            if (V == RV || at[u] >= 0) rope_store<V>(a[u], dst[u]);
            else rope_store<RV>(a[u], dst[u]);
        }
    }
}

}  // namespace enchip
