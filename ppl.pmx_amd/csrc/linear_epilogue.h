// Shared by the kernels of the linear with bias, activation and residual: the activations, their slopes, and
// what happens to eight neighbouring columns of H = X W^T once they are complete.
//   Y = act(H + B) + R, all in fp32 and rounded once.
#pragma once
#include "common.h"

namespace opmx {
namespace {

typedef uint32_t quad_any __attribute__((ext_vector_type(4), aligned(2)));     // 16 bytes at any address
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));

// The logistic function as in the SwiGLU kernels: accurate where the output keeps its digits.
template <typename T> __device__ __forceinline__ float logistic_for(float x)
{
    if constexpr (sizeof(T) == 2) return sigmoid_fast_(x);
    else return sigmoidf_(x);
}

constexpr float kSqrtHalf = 0.70710678118654752f, kGeluC = 0.79788456080286536f, kGeluA = 0.044715f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// erfc keeps its relative accuracy where 1 + erf would cancel (h < 0).
template <typename T> __device__ __forceinline__ float activate(int act, float h)
{
    switch (act) {
        case OPMX_ACTIVATION_SILU: return h * logistic_for<T>(h);
        case OPMX_ACTIVATION_GELU: return 0.5f * h * erfcf(-h * kSqrtHalf);
        case OPMX_ACTIVATION_GELU_TANH: return h * logistic_for<T>(2.0f * kGeluC * (h + kGeluA * h * h * h));
    }
    return h;
}
template <typename T> __device__ __forceinline__ float slope(int act, float h)
{
    switch (act) {
        case OPMX_ACTIVATION_SILU: {
            const float s = logistic_for<T>(h);
            return s + h * s * (1.0f - s);
        }
        case OPMX_ACTIVATION_GELU:
            return 0.5f * erfcf(-h * kSqrtHalf) + h * expf(-0.5f * h * h) * kInvSqrt2Pi;
        case OPMX_ACTIVATION_GELU_TANH: {
            const float s = logistic_for<T>(2.0f * kGeluC * (h + kGeluA * h * h * h));
            const float q = h * h;
            return s + h * s * (1.0f - s) * (2.0f * kGeluC * (1.0f + 3.0f * kGeluA * q));
        }
    }
    return 1.0f;
}

// Eight consecutive values of a row at any address; `left` of them exist.
template <typename T> __device__ __forceinline__ void load8(const T *p, int64_t left, float (&v)[8])
{
    constexpr int n = 16 / sizeof(T);
    if (left >= 8) {
#pragma unroll
        for (int c = 0; c < 8 / n; ++c) {
            T t[n];
            const quad_any q = *reinterpret_cast<const quad_any *>(p + c * n);
            __builtin_memcpy(t, &q, 16);
#pragma unroll
            for (int j = 0; j < n; ++j) v[c * n + j] = to_f32(t[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < left ? to_f32(p[j]) : 0.0f;
    }
}
template <typename T> __device__ __forceinline__ void store8(T *p, int64_t left, const float (&v)[8])
{
    constexpr int n = 16 / sizeof(T);
    if (left >= 8) {
#pragma unroll
        for (int c = 0; c < 8 / n; ++c) {
            T t[n];
#pragma unroll
            for (int j = 0; j < n; ++j) t[j] = from_f32<T>(v[c * n + j]);
            quad_any q;
            __builtin_memcpy(&q, t, 16);
            *reinterpret_cast<quad_any *>(p + c * n) = q;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = from_f32<T>(v[j]);
    }
}

// H = X W^T + B as it is kept for the backward pass: fp32 values as they are, in the 16-bit types as 24 bits of the fp32
// value, 16 in a first plane and the next 8 in a second one behind it.  In 16 bits the rounding of H alone would
// move the gradients as much as the rounding of dH for the matrix units does (bf16, SwiGLU: 0.0030 of their norm
// off instead of 0.0024); 24 bits cost one byte per value more to write and to read.
template <typename T> __device__ __forceinline__ void keep8(void *kept, int64_t count, int64_t at, int64_t left, const float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        store8(static_cast<float *>(kept) + at, left, v);
    } else {
        uint16_t *hi = static_cast<uint16_t *>(kept) + at;
        uint8_t *lo = reinterpret_cast<uint8_t *>(static_cast<uint16_t *>(kept) + count) + at;
        uint16_t a[8];
        uint8_t b[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = __float_as_uint(v[j]) + 0x80u;       // to nearest; infinities and NaNs stay what they are
            a[j] = static_cast<uint16_t>(u >> 16);
            b[j] = static_cast<uint8_t>(u >> 8);
        }
        if (left >= 8) {
            quad_any q;
            __builtin_memcpy(&q, a, 16);
            *reinterpret_cast<quad_any *>(hi) = q;
            __builtin_memcpy(lo, b, 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < left) {
                    hi[j] = a[j];
                    lo[j] = b[j];
                }
        }
    }
}
template <typename T> __device__ __forceinline__ void kept8(const void *kept, int64_t count, int64_t at, int64_t left, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        load8(static_cast<const float *>(kept) + at, left, v);
    } else {
        const uint16_t *hi = static_cast<const uint16_t *>(kept) + at;
        const uint8_t *lo = reinterpret_cast<const uint8_t *>(static_cast<const uint16_t *>(kept) + count) + at;
        uint16_t a[8];
        uint8_t b[8];
        if (left >= 8) {
            const quad_any q = *reinterpret_cast<const quad_any *>(hi);
            __builtin_memcpy(a, &q, 16);
            __builtin_memcpy(b, lo, 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                a[j] = j < left ? hi[j] : 0;
                b[j] = j < left ? lo[j] : 0;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = __uint_as_float((static_cast<uint32_t>(a[j]) << 16) | (static_cast<uint32_t>(b[j]) << 8));
    }
}

}  // namespace

// What a product's columns go through on their way out.
struct Epilogue {
    const void *bias = nullptr;       // [N]
    const void *residual = nullptr;   // [rows, ncols]
    void *Y = nullptr;                // [rows, ncols]
    void *H = nullptr;                // [rows, N] the sums with bias, for the backward pass (keep8)
    int64_t rows = 0, N = 0, ncols = 0;
    int act = OPMX_ACTIVATION_NONE;   // SWIGLU: ncols = N / 2
    float *part = nullptr;            // k ranges: fp32 sums [range][rows][pitch] instead of all of the above
    int64_t pitch = 0;
};

namespace {

// Columns col .. col+7 of row `row` (h; with SwiGLU h holds the first half's and g the second half's columns).
template <typename T, bool GATED>
__device__ __forceinline__ void finish8(const Epilogue &e, int64_t row, int64_t col, float (&h)[8], float (&g)[8])
{
    const int64_t left = e.ncols - col;
    if (left <= 0) return;
    if (e.bias) {
        float b[8];
        load8(static_cast<const T *>(e.bias) + col, left, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += b[j];
        if (GATED) {
            load8(static_cast<const T *>(e.bias) + e.ncols + col, left, b);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] += b[j];
        }
    }
    if (e.H) {
        keep8<T>(e.H, e.rows * e.N, row * e.N + col, left, h);
        if (GATED) keep8<T>(e.H, e.rows * e.N, row * e.N + e.ncols + col, left, g);
    }
    if (GATED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = g[j] * h[j] * logistic_for<T>(h[j]);
    } else if (e.act != OPMX_ACTIVATION_NONE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = activate<T>(e.act, h[j]);
    }
    if (e.residual) {
        float r[8];
        load8(static_cast<const T *>(e.residual) + row * e.ncols + col, left, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += r[j];
    }
    store8(static_cast<T *>(e.Y) + row * e.ncols + col, left, h);
}

}  // namespace

// C[m, c] = sum_k Q(m, k) P(c, k) over m < e.rows, c < e.N, and the epilogue.  An operand holds its rows one after
// the other in k (k_major false: element (r, k) at r * pitch + k) or its k values one after the other in rows
// (k_major true: at k * pitch + r).  16-byte aligned, pitch a multiple of 16 bytes; beyond that row counts and Kc
// are free where the values that fill up a chunk of 16 bytes may be read (they do not count).
struct Operand {
    const void *p;
    int64_t pitch;
    bool k_major;
};
// ranges > 1: k is cut into that many ranges, e.part must hold their sums.
int launch_linear_gemm(const Operand &P, const Operand &Q, int64_t Kc, int dtype, const Epilogue &e, int tile, int ranges,
                       hipStream_t s);

}  // namespace opmx
