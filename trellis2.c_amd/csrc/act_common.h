// act_common.h - the activations of epilogues.
#pragma once
#include <type_traits>

#include "tsh_internal.h"

namespace tsh {
namespace {

// For 16-bit outputs the hardware exponential and reciprocal (about 2^-21
// relative) stay far below the output's rounding; fp32 outputs of SiLU and of GELU
// with tanh take the accurate functions.  Both are v times a logistic function: of v,
// and of 2 sqrt(2 / pi) (v + 0.044715 v^3).
//
// GELU is v Phi(v), and below zero Phi is small beside 1: one minus an erf, or a
// polynomial that is right to some 1e-6 of 1, loses it.  16 bits: Phi(-a), a = |v|, is
// 2 to a polynomial, fitted to its logarithm for the least error of Phi, relative and
// absolute, as the output's rounding needs it, and falling beyond the fit so that the
// exponential is zero there.  bf16: degree 9, 2^-12.4 relative down to v = -13.2 (below
// that bf16 has no normal numbers for the result), 2^-20.2 absolute.  fp16: degree 7,
// 2^-16 relative down to -4.05, below that 2^-29.6 of GELU (half a step is 2^-25), 2^-21
// absolute.  14 instructions a value: 79,523 x 512 -> 2048 from 8-bit rows 181 us; with the
// form of fp32 below 184; as a logistic function of v R(v^2), which is 5.7e-6 off, 165.
// fp32: exp(-a^2 / 2) t Q(t), t = 1 / (1 + p a), as the tail falls like 1 / a beside the
// exponential; Q of degree 8, 2^-25.2 relative.  t, Q, their products and the exponential
// add some 16 roundings, the exponential's argument 1.5 a^2.
template <int DT> struct GeluTail {
    static constexpr int degree = 9;
    static constexpr float c[10] = {-0.999997854f,    -1.15119767f,    -0.458608121f,   -0.0538811572f,  0.00854993984f,
                                    -0.000976997311f, 7.58256283e-05f, -3.73059152e-06f, 1.03579488e-07f, -1.21999999e-09f};
};
template <> struct GeluTail<kF16> {
    static constexpr int degree = 7;
    static constexpr float c[8] = {-0.999998927f,  -1.15115595f,     -0.458844155f,   -0.0534294285f,
                                   0.00817629881f, -0.000829449506f, 4.70212144e-05f, -1.05048525e-06f};
};
template <> struct GeluTail<kF32> {
    static constexpr int degree = 8;
    static constexpr float p = 0.34f;
    static constexpr float c[9] = {0.135618851f, 0.136142388f,  0.11496748f,  0.116314463f, -0.0470853858f,
                                   0.205778807f, -0.276415288f, 0.141150713f, -0.0264720283f};
};
template <int DT> __device__ __forceinline__ float gelu(float v) {
    using G = GeluTail<DT>;
    float x = fabsf(v);
    if constexpr (DT == kF32) x = __builtin_amdgcn_rcpf(fmaf(G::p, x, 1.0f));
    float q = G::c[G::degree];
#pragma unroll
    for (int i = G::degree - 1; i >= 0; --i) q = fmaf(q, x, G::c[i]);
    float tail;
    if constexpr (DT == kF32) {
        tail = q * x * __builtin_amdgcn_exp2f(v * (v * -0.72134752f));
    } else {
        tail = __builtin_amdgcn_exp2f(q);
    }
    return v * (v > 0.0f ? 1.0f - tail : tail);
}
template <int DT, int ACT> __device__ __forceinline__ float activate(float v) {
    if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_SILU) {
        if constexpr (DT == kF32) return v / (1.0f + expf(-v));
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
    } else if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_GELU) {
        return gelu<DT>(v);
    } else if constexpr (ACT == TRELLIS_SPARSE_HIP_ACT_GELU_TANH) {
        // (1 + tanh(u)) / 2 = 1 / (1 + exp(-2u))
        const float r = 1.5957691216057308f + 0.0713548162726f * v * v;
        if constexpr (DT == kF32) return v / (1.0f + expf(-v * r));
        return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v * r));
    } else {
        return v;
    }
}

// f(the activation as a constant).
template <class F> __device__ __forceinline__ void by_act(int act, F && f) {
    switch (act) {
        case TRELLIS_SPARSE_HIP_ACT_SILU: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_SILU>()); break;
        case TRELLIS_SPARSE_HIP_ACT_GELU: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_GELU>()); break;
        case TRELLIS_SPARSE_HIP_ACT_GELU_TANH: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_GELU_TANH>()); break;
        default: f(std::integral_constant<int, TRELLIS_SPARSE_HIP_ACT_NONE>()); break;
    }
}

}  // namespace
}  // namespace tsh
