// gated.h -- the gate of a gated feed-forward block: act(g) * u on f32 pre-activations, in registers of the
// product's epilogue. 32768 x 4096 outputs of K = 1024 on MI355X, the W8A8 products alone, least and median of 24
// launches: 320 and 388 us with SiLU, 339 and 404 with GELU. The linears' GELU, its tails gathered in lists, took 595
// in a run in which this one took 397.
#pragma once

#include <hip/hip_runtime.h>

#pragma clang fp contract(off)

namespace enchip {

enum GateAct { GATE_SILU = 0, GATE_GELU = 1 };

// x / (1 + e^-x) within 4 ulp while it is above 2^-100: 2^z on the hardware with z = -x log2(e) and the rounding of z
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

// 0.5 x erfc(-x / sqrt 2), erfc(u) = t p(t) e^(-u^2) with t = 1 / (1 + 0.3275911 u) for u >= 0
// (Abramowitz and Stegun 7.1.26, the formula of erf_f32's tail: 1.5e-7 of 1) and 2 - erfc(-u) below:
// one path for every x, and nothing cancels where x is far negative. GELUF32's series near 0 is a
// little closer there; its list of tails costs more than this formula does.
__device__ __forceinline__ float gelu_gate_f32(float x) {
    const float u = fabsf(x) * 0.7071067811865476f;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, u, 1.0f));
    float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
    p = __builtin_fmaf(p, t, 1.421413741f);
    p = __builtin_fmaf(p, t, -0.284496736f);
    p = __builtin_fmaf(p, t, 0.254829592f);
    const float q = p * t * __builtin_amdgcn_exp2f(u * u * -1.4426950408889634f);
    return 0.5f * x * (x < 0.0f ? q : 2.0f - q);
}

__device__ __forceinline__ float gate_f32(int act, float g, float u) {  // act is uniform
    return (act == GATE_SILU ? silu_f32(g) : gelu_gate_f32(g)) * u;
}

}  // namespace enchip
