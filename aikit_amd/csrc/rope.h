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

// One thread per element pair or passed-through element; grid.y: rows.
template <bool INTERLEAVED>
__global__ __launch_bounds__(256) void rope_rows(const float *__restrict__ x, int64_t ldx, float *__restrict__ y,
                                                 int64_t ldy, const double *__restrict__ turns, float mscale,
                                                 const int32_t *__restrict__ pos, int64_t pos0, int64_t row0, int L,
                                                 int64_t rows, int heads, int hd, int r) {
    __shared__ float2 cs[ROPE_MAX_PAIRS];
    const int64_t row = blockIdx.x;
    const double p = pos ? (double)pos[row] : (double)(pos0 + (row0 + row) % L);
    for (int j = threadIdx.x; j < r / 2; j += 256) {
        const double t = p * turns[j];
        float s, c;
        sincospif(2.0f * (float)(t - rint(t)), &s, &c);
        cs[j] = make_float2(c * mscale, s * mscale);
    }
    __syncthreads();
    const float *xr = x + row * ldx;
    float *yr = y + row * ldy;
    const int ipr = r / 2 + (hd - r);
    for (int i = threadIdx.x; i < heads * ipr; i += 256) {
        const int h = i / ipr, e = i % ipr;
        if (e >= r / 2) {
            const int at = h * hd + r + (e - r / 2);
            yr[at] = xr[at];
            continue;
        }
        const int a = h * hd + (INTERLEAVED ? 2 * e : e), b = a + (INTERLEAVED ? 1 : r / 2);
        const float2 w = cs[e];
        const float x1 = xr[a], x2 = xr[b];
        yr[a] = x1 * w.x - x2 * w.y;
        yr[b] = x2 * w.x + x1 * w.y;
    }
}

}  // namespace enchip
