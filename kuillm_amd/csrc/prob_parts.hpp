// Attention probabilities as operands of 16-bit MFMAs, for the kernels that keep fp32's bits.
#pragma once

#include "common.hpp"

namespace kuiops {

// A probability p as a sum of 16-bit parts, one MFMA each, which keeps fp32's bits.
//   bf16: three parts, each the leading 8 bits of what is left, cut off: p exactly.
//   f16: two, rounded: 11 bits, and 11 of a remainder that has 12 and a sign: 2^-23 of
//   p is lost, and no more than half of f16's smallest step 2^-24 (see Shift).
template <typename T> struct Parts;
template <> struct Parts<bf16_t> {
    static constexpr int N = 3;
    static __device__ __forceinline__ float cut(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
    static __device__ __forceinline__ void split(float p, bf16_t (&x)[N]) {
        const float h = cut(p), r = p - h, m = cut(r);
        x[0] = (bf16_t)h;
        x[1] = (bf16_t)m;
        x[2] = (bf16_t)(r - m);
    }
};
template <> struct Parts<f16_t> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void split(float p, f16_t (&x)[N]) {
        x[0] = from_f32<f16_t>(p);
        x[1] = from_f32<f16_t>(p - to_f32(x[0]));
    }
};

template <typename T> struct Shift;       // probabilities are relative to 2^(maximum + value)
template <> struct Shift<bf16_t> { static constexpr float value = 0.f; };       // p <= 2^8 between rescales
// p <= 2^15, and the row's largest is 2^7 at least: f16's smallest step 2^-24 is 2^-39 to
// 2^-31 of it
template <> struct Shift<f16_t> { static constexpr float value = -7.f; };
constexpr float kSlack = 8.f;       // a row's maximum may grow by 2^8 before its sums are rescaled

}  // namespace kuiops
