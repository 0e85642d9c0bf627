// gated.h -- the gate of a gated feed-forward block: act(g) * u on f32 pre-activations.
#pragma once

#include <hip/hip_runtime.h>

#include "gelu_f32.h"

#pragma clang fp contract(off)

namespace enchip {

enum GateAct { GATE_SILU = 0, GATE_GELU = 1 };

// x / (1 + e^-x) within 4 ulp: 2^z on the hardware with z = -x log2(e) and the rounding of z
// put back as a factor, an approximate reciprocal (1 ulp). x is bounded for the exponent only:
// past +-150 e^-x is 0 or infinite in f32, so x = +inf gives +inf and x = -inf NaN, as the
// formula does.
__device__ __forceinline__ float silu_f32(float x) {
    const float xb = __builtin_amdgcn_fmed3f(x, -150.0f, 150.0f);
    const float z = xb * -1.4426950408889634f;
    // -xb log2(e) - z, log2(e) in two parts
    const float r = __builtin_fmaf(xb, -1.9259629911e-8f, __builtin_fmaf(xb, -1.4426950408889634f, -z));
    const float e = __builtin_amdgcn_exp2f(z) * __builtin_fmaf(r, 0.6931471805599453f, 1.0f);
    return x * __builtin_amdgcn_rcpf(1.0f + e);
}

// GELUF32 without branches: both sides of |u| = 1 are computed, the one that applies is taken.
__device__ __forceinline__ float gelu_f32_select(float x) {
    bool tail;
    const float s = gelu_f32_series(x, tail);
    const float t = gelu_f32_offseries(x);
    return tail ? t : s;
}

__device__ __forceinline__ float gate_f32(int act, float g, float u) {  // act is uniform
    return (act == GATE_SILU ? silu_f32(g) : gelu_f32_select(g)) * u;
}

}  // namespace enchip
