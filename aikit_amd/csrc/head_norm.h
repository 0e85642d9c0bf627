// head_norm.h -- RMS norms of query and key heads, with the position rotation in the same pass.
//
// A head x of hd elements becomes n = x / sqrt(mean(x^2) + eps) * gain (the query's or the key's), its
// first r elements then turned by the row's position as rope.h does: pair j of the layout by p f_j, times
// mscale. Elements from r on are the normed ones (r = 0: no rotation). Apart, the two passes would read and
// write the rows twice.
//
// The squares are summed in 64 bits (a value of 1e30 squared is past 32), and 1 / sqrt is taken there: the
// hardware's 2^-24 estimate and one Newton step. It is applied as a power of two and a factor in [1/2, 1),
// so that no finite head overflows or loses bits on the way. An element is within 5 2^-23 mscale
// (|n1| + |n2|) of the formula (rope.h's roundings and three more; 2^-22 |n| where it is not turned).
//
// G lanes hold a head: slot s of a head is two groups of V elements that belong together (the pair's two
// halves, or neighbours), lane g has slots g, g + G, .... A sum over the head is log2 G exchanges, and every
// element is loaded and stored once by one lane, in place or not. The angles of a workgroup's rows are
// computed once, into LDS, while the first rows are on their way.
//
// Bound by memory: 8 bytes an element. 64 x 512 rows of 24 heads of 64 (403 MB) take 75 us on MI355X, 5.4 TB/s (a
// large copy 4.9; norms and rotation in two passes of elementary operations 811); 20011 rows of 20 heads of 128 at
// positions of their own, interleaved, 89 us, 4.6 TB/s; 16 rows 5 us, a call's latency. Rows loaded after the angles
// took 82 and 92 us.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rope.h"

#pragma clang fp contract(off)

namespace enchip {

struct HeadNorm {
    const float *gain_q, *gain_k;  // [hd]
    double eps, inv_hd;
    int q_heads;  // heads from q_heads on are keys
    int hd, r;
    int slots, turned;  // slots of a head, the first `turned` of them rotated
    int lanes;          // G, a power of two up to 64
};

// IT: slots of a lane (slots <= IT * G); V-wide accesses are aligned: the launch chooses them so.
template <bool INTERLEAVED, int V, int IT>
__global__ __launch_bounds__(256) void head_norm_rope(const float *x, int64_t ldx, float *y, int64_t ldy, HeadNorm p,
                                                      const double2 *__restrict__ turns, float mscale,
                                                      const int32_t *__restrict__ pos, int64_t pos0, int64_t row0, int L,
                                                      int64_t rows, int TR, FastDiv heads) {
    constexpr int BATCH = IT >= 4 ? 1 : 4 / IT;  // heads of a lane group in flight together
    __shared__ float2 cs[ROPE_CS];
    const int64_t first = (int64_t)blockIdx.x * TR;
    const int tr = (int)min((int64_t)TR, rows - first), np = p.r / 2;
    const int G = p.lanes, g = threadIdx.x & (G - 1), groups = 256 / G, group = threadIdx.x / G;
    const int units = tr * (int)heads.d;  // heads of the workgroup's rows
    // the lane's slots: offsets of their two parts, the same for every head
    int oa[IT], ob[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int s = g + G * i;
        const bool turn = s < p.turned;
        oa[i] = s >= p.slots ? -1 : !turn ? p.r + 2 * V * (s - p.turned) : INTERLEAVED ? 2 * V * s : V * s;
        ob[i] = oa[i] < 0 ? -1 : turn && !INTERLEAVED ? oa[i] + np : oa[i] + V;
        if (ob[i] >= p.hd) ob[i] = -1;
    }
    float v[BATCH][IT][2 * V];
    auto load = [&](int u0) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int u = min(u0 + group + groups * b, units - 1);
            const int row = (int)heads.div((uint32_t)u), h = u - row * (int)heads.d;
            const float *src = x + (first + row) * ldx + (int64_t)h * p.hd;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
#pragma unroll
                for (int k = 0; k < 2 * V; ++k) v[b][i][k] = 0.0f;
                if (oa[i] >= 0) rope_load<V>(v[b][i], src + oa[i]);
                if (ob[i] >= 0) rope_load<V>(v[b][i] + V, src + ob[i]);
            }
        }
    };
    load(0);  // in flight while the angles are formed
    for (int t = threadIdx.x; t < tr * np; t += 256) {
        const int row = t / np, j = t - row * np;
        const double at = pos ? (double)pos[first + row] : (double)(pos0 + (row0 + first + row) % L);
        const double2 f = turns[j];
        const double a = at * f.x, e = __builtin_fma(at, f.y, __builtin_fma(at, f.x, -a));
        float s, c;
        sincospif(2.0f * (float)(a - rint(a) + e), &s, &c);
        cs[t] = make_float2(c * mscale, s * mscale);
    }
    float gq[IT][2 * V], gk[IT][2 * V];
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            gq[i][k] = oa[i] >= 0 ? p.gain_q[oa[i] + k] : 0.0f;
            gk[i][k] = oa[i] >= 0 ? p.gain_k[oa[i] + k] : 0.0f;
            gq[i][V + k] = ob[i] >= 0 ? p.gain_q[ob[i] + k] : 0.0f;
            gk[i][V + k] = ob[i] >= 0 ? p.gain_k[ob[i] + k] : 0.0f;
        }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    for (int u0 = 0; u0 < units; u0 += groups * BATCH) {  // uniform: the exchanges need every lane
        if (u0 > 0) load(u0);
        double sum[BATCH];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            sum[b] = 0.0;
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int k = 0; k < 2 * V; ++k) sum[b] = __builtin_fma((double)v[b][i][k], (double)v[b][i][k], sum[b]);
        }
        for (int o = G >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int b = 0; b < BATCH; ++b) sum[b] += __shfl_xor(sum[b], o, 64);
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int u = u0 + group + groups * b;
            if (u >= units) continue;
            const int row = (int)heads.div((uint32_t)u), h = u - row * (int)heads.d;
            const double ms = __builtin_fma(sum[b], p.inv_hd, p.eps);
            double rs = __builtin_amdgcn_rsq(ms);
            rs = rs * __builtin_fma(-0.5 * ms * rs, rs, 1.5);
            if (ms > 0x1p1000) rs = 0.0;  // an infinite element is NaN, the others 0, as the formula has them
            const int ex = __builtin_amdgcn_frexp_exp(rs);
            const float fr = (float)__builtin_amdgcn_frexp_mant(rs);
            const bool query = h < p.q_heads;
            float *dst = y + (first + row) * ldy + (int64_t)h * p.hd;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                float n[2 * V];
#pragma unroll
                for (int k = 0; k < 2 * V; ++k) n[k] = ldexpf(v[b][i][k], ex) * fr * (query ? gq[i][k] : gk[i][k]);
                if (g + G * i < p.turned) {
                    const float2 *w = cs + row * np + V * (g + G * i);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        constexpr bool INNER = INTERLEAVED && V > 1;
                        float &e1 = n[INNER ? 2 * k : k], &e2 = n[INNER ? 2 * k + 1 : V + k];
                        const float x1 = e1, x2 = e2;
                        e1 = x1 * w[k].x - x2 * w[k].y;
                        e2 = x2 * w[k].x + x1 * w[k].y;
                    }
                }
                if (oa[i] >= 0) rope_store<V>(n, dst + oa[i]);
                if (ob[i] >= 0) rope_store<V>(n + V, dst + ob[i]);
            }
        }
    }
}

}  // namespace enchip
