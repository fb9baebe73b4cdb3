// Activations kept in 8 bits for the backward pass (checkpoint8.h): pack and unpack of whole rows, and
// SwiGLU whose input is kept that way -- forward writes the output and the 8-bit input in one pass over X,
// backward reads the 8-bit input and dY and writes dX.
//   Y = g a s(beta a),  s the logistic function, X = (a | g)
//   dg = dY a s(beta a),  da = dY g s(beta a) (1 + beta a (1 - s(beta a)))      at the held a, g
// All of it is elementwise and bound by memory: [16384, 2 x 14336] bfloat16 moves 1.89 GB forward, in 343 us (5.5 TB/s), and as
// much backward, in 318 us (5.9 TB/s; a copy of that size reaches 4.9), from a replayed graph; pack and unpack of
// [16384, 14336] 134 and 126 us (5.3 and 5.7 TB/s).  A lane takes 16 bytes of a row, so a block of 32 values lies in
// 4 (16-bit types) or 8 (fp32) neighbouring lanes and its largest magnitude is two or three cross-lane steps.
// Rows may start at any address: loads and stores of 16 bytes need no alignment on this part, only the
// last values of a row that fill no chunk go one by one.
#include "checkpoint8.h"

#include <cfloat>
#include <type_traits>

namespace opmx {
namespace {

typedef uint32_t quad __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes at any address of a 16-bit value

template <typename T> struct Chunk {
    static constexpr int n = 16 / sizeof(T);
    T v[n];
};

// The chunk of up to n values at p (`left` of them exist, the others read as zero).
template <typename T> __device__ __forceinline__ Chunk<T> load_chunk(const T *p, int64_t left)
{
    Chunk<T> c;
    if (left >= Chunk<T>::n) {
        const quad q = __builtin_nontemporal_load(reinterpret_cast<const quad *>(p));
        __builtin_memcpy(&c, &q, 16);
    } else {
#pragma unroll
        for (int j = 0; j < Chunk<T>::n; ++j) c.v[j] = j < left ? p[j] : from_f32<T>(0.0f);
    }
    return c;
}
template <typename T> __device__ __forceinline__ void store_chunk(T *p, const Chunk<T> &c, int64_t left)
{
    if (left >= Chunk<T>::n) {
        quad q;
        __builtin_memcpy(&q, &c, 16);
        *reinterpret_cast<quad *>(p) = q;
    } else {
#pragma unroll
        for (int j = 0; j < Chunk<T>::n; ++j)
            if (j < left) p[j] = c.v[j];
    }
}

// The same chunk, of which the compiler knows nothing: what a rare branch works out of it is not held in registers before.
template <typename T> __device__ __forceinline__ Chunk<T> anew(Chunk<T> c)
{
    quad q;
    __builtin_memcpy(&q, &c, 16);
    asm volatile("" : "+v"(q));
    __builtin_memcpy(&c, &q, 16);
    return c;
}

// n bytes (8 or 4) at an address of any alignment.
template <int n> struct Bytes {
    signed char v[n];
};
template <int n> __device__ __forceinline__ Bytes<n> load_bytes(const int8_t *p, int64_t left)
{
    Bytes<n> b;
    if (left >= n) {
        __builtin_memcpy(&b, p, n);
    } else {
#pragma unroll
        for (int j = 0; j < n; ++j) b.v[j] = j < left ? p[j] : 0;
    }
    return b;
}
template <int n> __device__ __forceinline__ void store_bytes(int8_t *p, const Bytes<n> &b, int64_t left)
{
    if (left >= n) {
        __builtin_memcpy(p, &b, n);
    } else {
#pragma unroll
        for (int j = 0; j < n; ++j)
            if (j < left) p[j] = b.v[j];
    }
}

// Packs a lane's chunk; every lane of the wave takes part (lanes past the row hold zeros).  `lead` lanes write
// the block's code.
template <typename T>
__device__ __forceinline__ void pack_chunk(const Chunk<T> &x, int64_t left, int8_t *q, uint8_t *code_at)
{
    constexpr int n = Chunk<T>::n, lanes = kBlock8 / n;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < n; ++j) {
        const uint32_t b = __float_as_uint(to_f32(x.v[j])) & 0x7FFFFFFFu;
        m = b > m ? b : m;
    }
#pragma unroll
    for (int d = 1; d < lanes; d <<= 1) {
        const uint32_t o = __shfl_xor(m, d, kWave);
        m = o > m ? o : m;
    }
    const uint32_t code = step_code<T>(m);
    if (left > 0) {
        Bytes<n> b;
#pragma unroll
        for (int j = 0; j < n; ++j) b.v[j] = static_cast<int8_t>(to_steps(to_f32(x.v[j]), code));
        store_bytes<n>(q, b, left);
        if (threadIdx.x % lanes == 0) *code_at = static_cast<uint8_t>(code);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void pack8_kernel(const T *__restrict__ X, int64_t R, int64_t D, int64_t blocks,
                                                    int8_t *__restrict__ q, uint8_t *__restrict__ codes)
{
    constexpr int n = Chunk<T>::n;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * n, left = D - c;
    const int64_t step = static_cast<int64_t>(gridDim.y) * blockDim.y;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * blockDim.y; r0 < R; r0 += step) {
        const int64_t r = r0 + threadIdx.y, here = r < R ? left : 0;
        const Chunk<T> x = load_chunk(X + r * D + c, here);
        pack_chunk(x, here, q + r * D + c, codes + r * blocks + c / kBlock8);
    }
}

template <typename T>
__global__ __launch_bounds__(256) void unpack8_kernel(const int8_t *__restrict__ q, const uint8_t *__restrict__ codes,
                                                      int64_t R, int64_t D, int64_t blocks, int64_t pitch,
                                                      T *__restrict__ X)
{
    constexpr int n = Chunk<T>::n;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * n, left = D - c;
    if (left <= 0) return;
    const int64_t step = static_cast<int64_t>(gridDim.y) * blockDim.y;
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; r < R; r += step) {
        const uint32_t code = codes[r * blocks + c / kBlock8];
        const Bytes<n> b = load_bytes<n>(q + r * D + c, left);
        Chunk<T> x;
#pragma unroll
        for (int j = 0; j < n; ++j) x.v[j] = from_f32<T>(from_steps(b.v[j], code));
        store_chunk(X + r * pitch + c, x, left);
    }
}

// As for the plain SwiGLU kernel: the accurate logistic function where the output keeps its digits.
template <typename T> __device__ __forceinline__ float logistic(float x)
{
    if constexpr (sizeof(T) == 2) return sigmoid_fast_(x);
    else return sigmoidf_(x);
}

// The last product of the output, rounded as the plain operator does.  In float16 its form for whole 16-byte chunks rounds to fp32
// first and then to the type, its other form once (a value in 16000 differs); which instruction the compiler takes here
// would depend on what stands around it.
template <typename T, bool CHUNKS> __device__ __forceinline__ T last_product(float a, float b)
{
    if constexpr (!std::is_same<T, f16>::value) {
        return from_f32<T>(a * b);
    } else if constexpr (CHUNKS) {
        float p = a * b;
        asm("" : "+v"(p));
        return from_f32<T>(p);
    } else {
        uint32_t r;
        asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(r) : "v"(a), "v"(b));
        const uint16_t low = static_cast<uint16_t>(r);
        T v;
        __builtin_memcpy(&v, &low, 2);
        return v;
    }
}

// KEEP: q and codes are wanted.  CHUNKS: the plain operator would take this call 16 bytes at a time.
template <typename T, bool KEEP, bool CHUNKS>
__global__ __launch_bounds__(256) void swiglu8_kernel(const T *__restrict__ X, int64_t R, int64_t D, int64_t blocks,
                                                      float beta, T *__restrict__ Y, int8_t *__restrict__ q,
                                                      uint8_t *__restrict__ codes)
{
    constexpr int n = Chunk<T>::n;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * n, left = D - c;
    const int64_t step = static_cast<int64_t>(gridDim.y) * blockDim.y;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * blockDim.y; r0 < R; r0 += step) {
        const int64_t r = r0 + threadIdx.y, here = r < R ? left : 0;
        const Chunk<T> a = load_chunk(X + r * 2 * D + c, here), g = load_chunk(X + r * 2 * D + D + c, here);
        Chunk<T> y;
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const float af = to_f32(a.v[j]), ga = to_f32(g.v[j]) * af;
            most = fmaxf(most, fabsf(ga));
            y.v[j] = last_product<T, CHUNKS>(ga, logistic<T>(beta * af));
        }
        // some g a is beyond fp32 (which it cannot be in float16): there a s first
        if (!std::is_same<T, f16>::value && most == INFINITY) {
            const Chunk<T> a2 = anew(a), g2 = anew(g);
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const float af = to_f32(a2.v[j]), gf = to_f32(g2.v[j]), s = logistic<T>(beta * af);
                if (fabsf(gf * af) == INFINITY) y.v[j] = from_f32<T>(gf * (af * s));
            }
        }
        store_chunk(Y + r * D + c, y, here);
        if constexpr (KEEP) {
            pack_chunk(a, here, q + r * 2 * D + c, codes + r * 2 * blocks + c / kBlock8);
            pack_chunk(g, here, q + r * 2 * D + D + c, codes + (r * 2 + 1) * blocks + c / kBlock8);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void swiglu8_backward_kernel(const T *__restrict__ dY, const int8_t *__restrict__ q,
                                                               const uint8_t *__restrict__ codes, int64_t R, int64_t D,
                                                               int64_t blocks, float beta, T *__restrict__ dX)
{
    constexpr int n = Chunk<T>::n;
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * n, left = D - c;
    if (left <= 0) return;
    const int64_t step = static_cast<int64_t>(gridDim.y) * blockDim.y;
    // `here` values exist: a constant where all do, so that nothing stands between the loads (7 % slower without)
    auto rows = [&](auto here) {
        for (int64_t r = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; r < R; r += step) {
            const uint32_t ca = codes[r * 2 * blocks + c / kBlock8], cg = codes[(r * 2 + 1) * blocks + c / kBlock8];
            const Bytes<n> qa = load_bytes<n>(q + r * 2 * D + c, here), qg = load_bytes<n>(q + r * 2 * D + D + c, here);
            const Chunk<T> dy = load_chunk(dY + r * D + c, here);
            Chunk<T> da, dg;
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const float a = from_steps(qa.v[j], ca), g = from_steps(qg.v[j], cg), d = to_f32(dy.v[j]);
                const float s = logistic<T>(beta * a);
                // The factors of d are finite where a and g are; d a and d g alone may overflow where s is 0.  Where beta a
                // overflows, s is 0 or 1 and any finite value serves for it.
                const float ba = __builtin_amdgcn_fmed3f(beta * a, -FLT_MAX, FLT_MAX);
                dg.v[j] = from_f32<T>(d * (a * s));
                da.v[j] = from_f32<T>(d * (g * (s + ba * s * (1.0f - s))));
            }
            store_chunk(dX + r * 2 * D + c, da, here);
            store_chunk(dX + r * 2 * D + D + c, dg, here);
        }
    };
    if (left >= n) rows(std::integral_constant<int, n>{});
    else rows(left);
}

// Blocks of 256 lanes over a strip of a row, or over several rows where rows are short; the lanes of a
// block of 32 values never straddle two rows of lanes (blockDim.x is a power of two >= 8).
struct Shape {
    dim3 grid, block;
};
template <typename T> inline Shape shape_for(int64_t R, int64_t D)
{
    constexpr int n = Chunk<T>::n;
    const int64_t lanes = ceil_div(D, kBlock8) * (kBlock8 / n);
    int bx = 8;
    while (bx < 256 && bx < lanes) bx <<= 1;
    const int by = 256 / bx;
    const int64_t rows = ceil_div(R, by);
    return {dim3(static_cast<unsigned>(ceil_div(lanes, bx)), static_cast<unsigned>(rows < 65535 ? rows : 65535)),
            dim3(bx, by)};
}

template <typename T> int pack8_impl(const void *X, int64_t R, int64_t D, void *q, void *codes, hipStream_t s)
{
    const Shape g = shape_for<T>(R, D);
    pack8_kernel<T><<<g.grid, g.block, 0, s>>>(static_cast<const T *>(X), R, D, ceil_div(D, kBlock8),
                                               static_cast<int8_t *>(q), static_cast<uint8_t *>(codes));
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}
template <typename T>
int unpack8_impl(const void *q, const void *codes, int64_t R, int64_t D, int64_t pitch, void *X, hipStream_t s)
{
    const Shape g = shape_for<T>(R, D);
    unpack8_kernel<T><<<g.grid, g.block, 0, s>>>(static_cast<const int8_t *>(q), static_cast<const uint8_t *>(codes), R, D,
                                                 ceil_div(D, kBlock8), pitch, static_cast<T *>(X));
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}
template <typename T>
int swiglu8_impl(const void *X, int64_t R, int64_t D, float beta, void *Y, void *q, void *codes, hipStream_t s)
{
    const Shape g = shape_for<T>(R, D);
    auto launch = [&](auto keep, auto chunks) {
        swiglu8_kernel<T, decltype(keep)::value, decltype(chunks)::value><<<g.grid, g.block, 0, s>>>(
            static_cast<const T *>(X), R, D, ceil_div(D, kBlock8), beta, static_cast<T *>(Y), static_cast<int8_t *>(q),
            static_cast<uint8_t *>(codes));
    };
    bool chunks = false;
    if constexpr (std::is_same<T, f16>::value) {
        chunks = D % Chunk<T>::n == 0 && aligned16(X) && aligned16(Y);
        if (chunks && q) launch(std::true_type{}, std::true_type{});
        else if (chunks) launch(std::false_type{}, std::true_type{});
    }
    if (!chunks && q) launch(std::true_type{}, std::false_type{});
    else if (!chunks) launch(std::false_type{}, std::false_type{});
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}
template <typename T>
int swiglu8_backward_impl(const void *dY, const void *q, const void *codes, int64_t R, int64_t D, float beta, void *dX,
                          hipStream_t s)
{
    const Shape g = shape_for<T>(R, D);
    swiglu8_backward_kernel<T><<<g.grid, g.block, 0, s>>>(static_cast<const T *>(dY), static_cast<const int8_t *>(q),
                                                          static_cast<const uint8_t *>(codes), R, D,
                                                          ceil_div(D, kBlock8), beta, static_cast<T *>(dX));
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

}  // namespace

int launch_checkpoint8_pack(const void *X, int64_t R, int64_t D, int dtype, void *q, void *codes, hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return pack8_impl<float>(X, R, D, q, codes, s);
        case OPMX_DTYPE_F16: return pack8_impl<f16>(X, R, D, q, codes, s);
        case OPMX_DTYPE_BF16: return pack8_impl<bf16>(X, R, D, q, codes, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

int launch_checkpoint8_unpack(const void *q, const void *codes, int64_t R, int64_t D, int dtype, void *X, hipStream_t s,
                              int64_t pitch)
{
    if (R == 0 || D == 0) return OPMX_OK;
    if (pitch == 0) pitch = D;
    switch (dtype) {
        case OPMX_DTYPE_F32: return unpack8_impl<float>(q, codes, R, D, pitch, X, s);
        case OPMX_DTYPE_F16: return unpack8_impl<f16>(q, codes, R, D, pitch, X, s);
        case OPMX_DTYPE_BF16: return unpack8_impl<bf16>(q, codes, R, D, pitch, X, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

int launch_swiglu_checkpoint8(const void *X, int64_t R, int64_t D, float beta, int dtype, void *Y, void *q, void *codes,
                              hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return swiglu8_impl<float>(X, R, D, beta, Y, q, codes, s);
        case OPMX_DTYPE_F16: return swiglu8_impl<f16>(X, R, D, beta, Y, q, codes, s);
        case OPMX_DTYPE_BF16: return swiglu8_impl<bf16>(X, R, D, beta, Y, q, codes, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

int launch_swiglu_checkpoint8_backward(const void *dY, const void *q, const void *codes, int64_t R, int64_t D, float beta,
                                       int dtype, void *dX, hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return swiglu8_backward_impl<float>(dY, q, codes, R, D, beta, dX, s);
        case OPMX_DTYPE_F16: return swiglu8_backward_impl<f16>(dY, q, codes, R, D, beta, dX, s);
        case OPMX_DTYPE_BF16: return swiglu8_backward_impl<bf16>(dY, q, codes, R, D, beta, dX, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

}  // namespace opmx
