// The 8-bit form in which activations are kept for a backward pass, shared by the kernels that
// write it and the ones that read it.
//
// Blocks of 32 consecutive values of a row (the last block of a row may be shorter) share a
// power-of-two step.  With m the largest magnitude of the block and 2^e the largest power of two not
// above m -- one more if m >= 1.9921875 * 2^e = 127.5 / 64 * 2^e, where round(m / step) would be 128, but
// never beyond the type's largest exponent -- the step is 2^max(e - 6, -126), a value x is held as the whole
// number round-half-even(x / step) in [-127, 127], and the block's code is the step's biased exponent, one
// byte.  Dividing by the step, rounding and multiplying back are exact in fp32, so every kernel agrees on
// every bit; |x - held(x)| <= max(m / 127.5, 2^-127): half a step, except that values beyond 127.5 steps at the very top
// of the type's range, where the step may not grow, are off by up to one, which is no more of m; and 2^-127 is
// half of the smallest step, so that a block below it is held as zeros.  A whole number of 7 bits times
// a power of two is exact in bfloat16 as well.  A block with an infinity or a NaN has code 255 and stands for
// NaN throughout: there is no step for it, and nothing finite may come out of it.
#pragma once
#include "train.h"

namespace opmx {
namespace {

constexpr int kBlock8 = 32;
constexpr uint32_t kNoStep = 255;

// Largest biased exponent of T: finite values of the type stay finite when read back.
template <typename T> struct MaxExponent { static constexpr uint32_t v = 254; };
template <> struct MaxExponent<f16> { static constexpr uint32_t v = 142; };

// Code of a block whose largest magnitude has the bits m (sign cleared; infinities and NaN compare larger).
template <typename T> __device__ __forceinline__ uint32_t step_code(uint32_t m)
{
    if (m >= 0x7F800000u) return kNoStep;
    uint32_t e = (m + 0x10000u) >> 23;          // + 2^-7 of the mantissa: carries from 1.9921875 on
    e = e < MaxExponent<T>::v ? e : MaxExponent<T>::v;
    return e > 7u ? e - 6u : 1u;
}
__device__ __forceinline__ float to_steps(float x, uint32_t code)
{
    if (code == kNoStep) return 0.0f;
    const float q = rintf(x * __uint_as_float((254u - code) << 23));   // 1 / step, exact
    return fminf(fmaxf(q, -127.0f), 127.0f);
}
__device__ __forceinline__ float from_steps(int q, uint32_t code)
{
    return code == kNoStep ? __uint_as_float(0x7FC00000u) : static_cast<float>(q) * __uint_as_float(code << 23);
}

}  // namespace
}  // namespace opmx
