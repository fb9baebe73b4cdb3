// Shared by the kernels of the linear with bias, activation and residual: the activations, their slopes, and
// what happens to eight neighbouring columns of H = X W^T once they are complete.
//   Y = act(H + B) + R, all in fp32 and rounded once.
#pragma once
#include "train.h"

namespace opmx {
namespace {

typedef uint32_t quad_any __attribute__((ext_vector_type(4), aligned(2)));     // 16 bytes at any address
typedef uint32_t pair_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));

// The logistic function as in the SwiGLU kernels: accurate where the output keeps its digits.
template <typename T> __device__ __forceinline__ float logistic_for(float x)
{
    if constexpr (sizeof(T) == 2) return sigmoid_fast_(x);
    else return sigmoidf_(x);
}

constexpr float kGeluC = 0.79788456080286536f, kGeluA = 0.044715f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// Phi(h) for GELU, and e^(-h^2 / 2), which the slope needs as well.  With z = |h| / sqrt 2, erfc(z) = e^(-z^2) t S(t) where
// t = 1 / (1 + 0.4 z) and S is smooth: a polynomial of degree 8 fitted to scipy's erfcx for z <= 14 (beyond,
// e^(-z^2) is 0 in fp32) is within 1.13e-7 of it, relatively, on both sides: Phi keeps its digits where it is small.
// In fp32 the whole is within 7e-7 (1 + h^2 / 4).  The library's erfc costs four times the instructions, in an epilogue
// whose time no matrix instruction hides.
__device__ __forceinline__ float normal_cdf(float h, float &bell)
{
    constexpr float kHalf[9] = {0.5f * 0.22566290199756622f, 0.5f * 0.22593672573566437f, 0.5f * 0.20561064779758453f,
                                0.5f * 0.17847903072834015f, 0.5f * 0.11547110229730606f, 0.5f * 0.035431284457445145f,
                                0.5f * 0.13050033152103424f, 0.5f * -0.16306036710739136f, 0.5f * 0.0459684394299984f};
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.28284271247461901f * fabsf(h));
    float s = kHalf[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) s = s * t + kHalf[i];
    bell = __builtin_amdgcn_exp2f(h * h * -0.72134752044448170f);
    const float tail = bell * t * s;
    return h < 0.0f ? tail : 1.0f - tail;
}

template <typename T> __device__ __forceinline__ float activate(int act, float h)
{
    if (act == OPMX_ACTIVATION_GELU) {
        float bell;
        return h * normal_cdf(h, bell);
    }
    // silu and the tanh form of gelu are h s(x)
    const float x = act == OPMX_ACTIVATION_SILU ? h : 2.0f * kGeluC * (h + kGeluA * h * h * h);
    return h * logistic_for<T>(x);
}
template <typename T> __device__ __forceinline__ float slope(int act, float h)
{
    if (act == OPMX_ACTIVATION_GELU) {
        float bell;
        const float cdf = normal_cdf(h, bell);
        return cdf + h * bell * kInvSqrt2Pi;
    }
    const bool silu = act == OPMX_ACTIVATION_SILU;
    const float s = logistic_for<T>(silu ? h : 2.0f * kGeluC * (h + kGeluA * h * h * h));
    // The factor of the tanh form overflows from |h| = 2e19 on, and infinity times a 1 - s or an s of 0 is NaN.  From |h| = 11 on s is 0
    // or 1 exactly and any finite factor does: that of 32.
    const float b = fminf(fabsf(h), 32.0f);
    const float dx = silu ? 1.0f : 2.0f * kGeluC * (1.0f + 3.0f * kGeluA * b * b);
    return s + h * s * (1.0f - s) * dx;
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
        // (a load under a condition of its own would be waited for before the next: the first value stands in for those
        // that do not exist)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        if (left > 0) {
            T t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = p[j < left ? j : 0];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < left ? to_f32(t[j]) : 0.0f;
        }
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
            // to nearest, but the last finite values not up to infinity; infinities and NaNs stay what they are
            const uint32_t bits = __float_as_uint(v[j]), u = (bits & 0x7FFFFFFFu) < 0x7F7FFF80u ? bits + 0x80u : bits;
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
            const quad_any q = __builtin_nontemporal_load(reinterpret_cast<const quad_any *>(hi));
            const pair_any u = __builtin_nontemporal_load(reinterpret_cast<const pair_any *>(lo));
            __builtin_memcpy(a, &q, 16);
            __builtin_memcpy(b, &u, 8);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                a[j] = hi[j < left ? j : 0];            // left > 0; what does not exist is not used
                b[j] = lo[j < left ? j : 0];
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

// Columns col .. col+7 of row `row` (h; with SwiGLU h holds the first half's and g the second half's columns): bias,
// what is kept, activation.  The result is in h.
template <typename T, bool GATED>
__device__ __forceinline__ void activate8(const Epilogue &e, int64_t row, int64_t col, int64_t left, const float (&bh)[8],
                                          const float (&bg)[8], float (&h)[8], float (&g)[8])
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        h[j] += bh[j];
        if (GATED) g[j] += bg[j];
    }
    if (e.H) {
        keep8<T>(e.H, e.rows * e.N, row * e.N + col, left, h);
        if (GATED) keep8<T>(e.H, e.rows * e.N, row * e.N + e.ncols + col, left, g);
    }
    if (GATED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = g[j] * (h[j] * logistic_for<T>(h[j]));     // (g h alone may overflow where s is 0)
    } else if (e.act != OPMX_ACTIVATION_NONE) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = activate<T>(e.act, h[j]);
    }
}
template <typename T, bool GATED>
__device__ __forceinline__ void load_bias8(const Epilogue &e, int64_t col, float (&bh)[8], float (&bg)[8])
{
#pragma unroll
    for (int j = 0; j < 8; ++j) bh[j] = bg[j] = 0.0f;
    if (e.bias == nullptr || col >= e.ncols) return;
    load8(static_cast<const T *>(e.bias) + col, e.ncols - col, bh);
    if (GATED) load8(static_cast<const T *>(e.bias) + e.ncols + col, e.ncols - col, bg);
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
// Tiles of C: 256 x 256 by four waves of 128 x 128 (16-bit types, k in one range); 128 x 128 with two k-tiles in LDS, 64 x 128
// and (fp32) 32 x 128 with three, each by four waves and two workgroups to a CU.
enum class Tile { k256, k128, k64, k32 };
// ranges > 1: k is cut into that many ranges, e.part must hold their sums.
int launch_linear_gemm(const Operand &P, const Operand &Q, int64_t Kc, int dtype, const Epilogue &e, Tile tile, int ranges,
                       hipStream_t s);

// The product and its epilogue for up to 64 rows of X, from W and X as they are; and the microseconds that it takes, about.
double linear_few_rows_us(int64_t T, int64_t K, int64_t N, int dtype, bool gated);
int launch_linear_few_rows(const void *X, const void *W, int64_t K, int dtype, const Epilogue &e, hipStream_t s);

}  // namespace opmx
