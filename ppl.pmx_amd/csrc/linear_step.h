// A step of 16 bytes per lane on the matrix units for the linear's kernels: 32 values of k in the 16-bit types, 16 in fp32.
#pragma once
#include "moe_gemm.h"

#define OPMX_LDS(p) ((void __attribute__((address_space(3))) *)(p))

namespace opmx {
namespace {

template <typename T> struct Step;
template <> struct Step<f16> {
    using frag = half8_t;
    static __device__ __forceinline__ float4_t mma(frag p, frag q, float4_t c) { return Mfma<f16>::m16(p, q, c); }
};
template <> struct Step<bf16> {
    using frag = bf16x8_t;
    static __device__ __forceinline__ float4_t mma(frag p, frag q, float4_t c) { return Mfma<bf16>::m16(p, q, c); }
};
template <> struct Step<float> {
    using frag = float4_t;
    static __device__ __forceinline__ float4_t mma(frag p, frag q, float4_t c)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p[j], q[j], c, 0, 0, 0);
        return c;
    }
};

}  // namespace
}  // namespace opmx
