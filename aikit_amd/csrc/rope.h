// rope.h -- rotary positions on rows of heads.
//
// Row t at position p, pair j < r/2 of every head (freq f_j, mscale m):
//   (y1, y2) = m (x1 cos(p f_j) - x2 sin(p f_j), x2 cos(p f_j) + x1 sin(p f_j)),
// the pair being elements (j, j + r/2) of the head (half) or (2j, 2j + 1) (interleaved);
// elements r .. head_dim pass through.
//
// The angle is formed in turns, p f_j / 2 pi, in 64 bits and reduced there (a far position times
// a frequency keeps no fraction in 32), sine and cosine of the reduced angle in 32: an error of
// about 2^-23 of the pair's length at any position. The pairs' angles are those of every head of
// the row, so a workgroup computes them once for its rows into LDS and then streams the rows.
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
struct RopeVec {
    float v[V];
    __device__ __forceinline__ void load(const float *p) {
        if constexpr (V == 4) {
            const f32x4 t = *reinterpret_cast<const f32x4 *>(p);
            v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(float *p) const {
        if constexpr (V == 4) {
            *reinterpret_cast<f32x4 *>(p) = f32x4{v[0], v[1], v[2], v[3]};
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] = v[i];
        }
    }
};

// A workgroup's TR rows, as items of V elements: per head first the items of the rotated part (half:
// V elements of each half; interleaved: V elements, V / 2 pairs; V = 1: one pair), then, not in
// place, those of the passed-through part. ipr: items per head. V = 4: r a multiple of 8 (half) or
// 4, head_dim and pitches of 4, 16-byte aligned buffers.
template <bool INTERLEAVED, int V>
__global__ __launch_bounds__(256) void rope_rows(const float *x, int64_t ldx, float *y,
                                                 int64_t ldy, const double *__restrict__ turns, float mscale,
                                                 const int32_t *__restrict__ pos, int64_t pos0, int64_t row0, int L,
                                                 int64_t rows, int TR, FastDiv heads, FastDiv ipr, int hd, int r) {
    __shared__ float2 cs[ROPE_CS];
    constexpr int PV = INTERLEAVED && V == 4 ? 2 : 1;     // an item's pairs over V
    const int64_t first = (int64_t)blockIdx.x * TR;
    const int tr = (int)min((int64_t)TR, rows - first), np = r / 2;
    for (int t = threadIdx.x; t < tr * np; t += 256) {
        const int row = t / np, j = t - row * np;
        const double p = pos ? (double)pos[first + row] : (double)(pos0 + (row0 + first + row) % L);
        const double a = p * turns[j];
        float s, c;
        sincospif(2.0f * (float)(a - rint(a)), &s, &c);
        cs[t] = make_float2(c * mscale, s * mscale);
    }
    __syncthreads();
    const int rot = PV == 2 ? r / 4 : np / V;  // rotated items of a head
    const uint32_t items = (uint32_t)tr * heads.d * ipr.d;
    for (uint32_t i0 = threadIdx.x; i0 < items; i0 += 256 * ROPE_BATCH) {
        RopeVec<V> a[ROPE_BATCH], b[ROPE_BATCH];
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
            const int off = h * hd + (turn ? (INTERLEAVED ? (V == 4 ? 4 : 2) * e : V * e) : r + V * (e - rot));
            const float *src = x + (first + row) * ldx + off;
            dst[u] = y + (first + row) * ldy + off;
            at[u] = turn ? (int)row * np + (PV == 2 ? 2 : V) * e : -1;
            a[u].load(src);
            if (V == 1 ? turn : (!INTERLEAVED && turn)) b[u].load(src + (INTERLEAVED ? 1 : np));
        }
#pragma unroll
        for (int u = 0; u < ROPE_BATCH; ++u) {
            if (at[u] == -2) continue;
            if (at[u] >= 0) {
                if constexpr (PV == 2) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float2 w = cs[at[u] + k];
                        const float x1 = a[u].v[2 * k], x2 = a[u].v[2 * k + 1];
                        a[u].v[2 * k] = x1 * w.x - x2 * w.y;
                        a[u].v[2 * k + 1] = x2 * w.x + x1 * w.y;
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float2 w = cs[at[u] + k];
                        const float x1 = a[u].v[k], x2 = b[u].v[k];
                        a[u].v[k] = x1 * w.x - x2 * w.y;
                        b[u].v[k] = x2 * w.x + x1 * w.y;
                    }
                    b[u].store(dst[u] + (INTERLEAVED ? 1 : np));
                }
            }
            a[u].store(dst[u]);
        }
    }
}

}  // namespace enchip
