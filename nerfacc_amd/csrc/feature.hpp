// feature.hpp — what the feature operators (dense.hip, conv.hip, selective.hip) share: the three element types, activations with
// their derivatives, and the reduction of partial sums.
#pragma once

#include <utility>

#include "common.hpp"

namespace nfa {

constexpr int64_t kMaxThreads = 1ll << 32;   // of a launch, along one axis of its grid

using bf16 = __bf16;
using f16 = _Float16;

template <class T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
// one rounding to nearest even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32)
template <class T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

inline int64_t dtype_bytes(int32_t dtype) { return dtype == NFA_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int32_t dtype) { return dtype >= NFA_DTYPE_F32 && dtype <= NFA_DTYPE_F16; }

// calls f(T{}) with the element type of `dtype`
template <class F>
inline void with_dtype(int32_t dtype, F &&f) {
    if (dtype == NFA_DTYPE_F32) f(float{});
    else if (dtype == NFA_DTYPE_BF16) f(bf16{});
    else f(f16{});
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// 2^x in one v_exp_f32: 1 ulp, results below 2^-126 become 0
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// v_rcp_f32 (1 ulp)
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// sigmoid with the exponential taken of -|x|: no overflow at either end.  The relative error is a few ulp at x > 0; below, the rounding of the
// exponent adds 1.3 |x| 2^-24 (32 ulp at x = -80), and results below 2^-126 become 0
__device__ __forceinline__ float sigmoid_f(float x) {
    const float e = fast_exp2(-fabsf(x) * kLog2e), r = fast_rcp(1.0f + e);
    return x >= 0.0f ? r : e * r;                            // (NaN: e and r are)
}

// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1], with log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3, as its odd
// series: every term is positive, so small steps (x around -7 in a scan) keep their relative accuracy, which log(1 + e) would not.
// The series is cut after s^15 / 15: the rest is below (9 / 8) 3^-16 / 17 = 1.6e-9 of the first term.
__device__ __forceinline__ float softplus_from(float x, float e) {         // e = exp(-|x|)
    const float s = e * fast_rcp(2.0f + e), q = s * s;
    float p = 1.0f / 15.0f;
    p = fmaf(p, q, 1.0f / 13.0f);
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    p = fmaf(p, q, 1.0f);
    return fmaf(s + s, p, fmaxf(x, 0.0f));                   // (NaN: s is)
}
__device__ __forceinline__ float softplus_f(float x) { return softplus_from(x, fast_exp2(-fabsf(x) * kLog2e)); }

constexpr float kInvSqrt2 = 0.70710678118654752f, kInvSqrt2Pi = 0.39894228040143268f;

// What a layer keeps for its backward pass (include/nerfacc_hip.h: nfa_linear_saved_bytes).  relu: one bit, or its value.  The others, by type:
//   fp32  the number that act' comes from in full: a = act(z) for exp and softplus (a itself; 1 - e^-a, as accurate as a), else z;
//   bf16  act' rounded once, so that its relative error is bf16's at any z (z kept in bf16 would lose |z| times that where act' decays:
//         6 % of sigmoid' at z = -16); a for exp and softplus, which round alike;
//   fp16  act' in 32 bits: below z = -10 sigmoid', softplus' and exp' are under 2^-14, where fp16 has fewer and fewer bits.
constexpr bool act_from_value(int32_t act) { return act == NFA_ACT_RELU || act == NFA_ACT_EXP || act == NFA_ACT_SOFTPLUS; }

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
    if constexpr (ACT == NFA_ACT_RELU) return z < 0.0f ? 0.0f : z;      // (NaN stays NaN)
    else if constexpr (ACT == NFA_ACT_SIGMOID) return sigmoid_f(z);
    else if constexpr (ACT == NFA_ACT_SOFTPLUS) return softplus_f(z);
    else if constexpr (ACT == NFA_ACT_SILU) return z * sigmoid_f(z);
    else if constexpr (ACT == NFA_ACT_GELU) return 0.5f * z * erfcf(-z * kInvSqrt2);
    else if constexpr (ACT == NFA_ACT_EXP) return expf(z);
    else return z;
}
// the derivative of a smooth activation, from z
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if constexpr (ACT == NFA_ACT_SIGMOID) return sigmoid_f(z) * sigmoid_f(-z);
    else if constexpr (ACT == NFA_ACT_SOFTPLUS) return sigmoid_f(z);
    else if constexpr (ACT == NFA_ACT_SILU) return sigmoid_f(z) * fmaf(z, sigmoid_f(-z), 1.0f);
    else if constexpr (ACT == NFA_ACT_GELU) return fmaf(z * kInvSqrt2Pi, expf(-0.5f * z * z), 0.5f * erfcf(-z * kInvSqrt2));
    else return expf(z);
}
// the same from what fp32 keeps: the value of exp and softplus, z of the others
template <int ACT>
__device__ __forceinline__ float act_slope_of_kept(float s) {
    if constexpr (ACT == NFA_ACT_SOFTPLUS) return -expm1f(-s);
    else if constexpr (ACT == NFA_ACT_EXP) return s;
    else return act_slope<ACT>(s);
}
// calls f(integral ACT): the choice is made once around a loop, not once per number (a switch inside an unrolled loop is many times
// the instruction cache)
template <class F>
__device__ __forceinline__ void with_act(int act, F &&f) {
    switch (act) {
        case NFA_ACT_RELU: f(std::integral_constant<int, NFA_ACT_RELU>{}); break;
        case NFA_ACT_SIGMOID: f(std::integral_constant<int, NFA_ACT_SIGMOID>{}); break;
        case NFA_ACT_SOFTPLUS: f(std::integral_constant<int, NFA_ACT_SOFTPLUS>{}); break;
        case NFA_ACT_SILU: f(std::integral_constant<int, NFA_ACT_SILU>{}); break;
        case NFA_ACT_GELU: f(std::integral_constant<int, NFA_ACT_GELU>{}); break;
        case NFA_ACT_EXP: f(std::integral_constant<int, NFA_ACT_EXP>{}); break;
        default: f(std::integral_constant<int, NFA_ACT_NONE>{}); break;
    }
}

inline bool act_ok(int32_t act) { return act >= NFA_ACT_NONE && act <= NFA_ACT_EXP; }

// the sum over the rows of part [rows][all columns] in a fixed order (no atomics: the same bits every time), rounded once; the columns
// go to up to three outputs (pointer or nullptr, columns), one behind the other.  part is written to.
void launch_reduce_rows(float *part, int64_t rows, std::initializer_list<std::pair<void *, int64_t>> outputs, int32_t dtype, hipStream_t s);

// n numbers of a type (pointer or nullptr): zeros, where a gradient has no rows to be summed over
void launch_zero(void *p, int64_t n, int32_t dtype, hipStream_t s);

}  // namespace nfa
