// Linear with bias, activation and residual in its epilogue: Y = act(X W^T + B) + R, and its gradients
//   dH = dY * act'(H),  dX = dH W,  dW = dH^T X,  dB = sum_t dH   (dR = dY).
// The products run in linear_gemm.hip; here are the passes around them and the choice of tiles.
//   pad         operands whose rows are not whole 16-byte chunks are copied to rows that are (the copy is
//               (T + N) K values against 2 T N K operations)
//   slope       dH from dY and the kept H in one pass, with the column sums for dB
//   join        products with few tiles are cut along k; the fp32 sums of the ranges meet here, in order, and
//               go through the epilogue
// dH is rounded to the tensors' type for the matrix units; H is kept with 16 bits of mantissa (keep8).
#include "checkpoint8.h"
#include "linear_epilogue.h"

#include <algorithm>
#include <type_traits>

namespace opmx {
namespace {

inline int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// X [R, C] dense -> [R][pitch], zeros behind the C values.
// Two tensors of the same C in one launch (blockIdx.z).
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T *__restrict__ X0, int64_t R0, T *__restrict__ out0,
                                                  const T *__restrict__ X1, int64_t R1, T *__restrict__ out1, int64_t C,
                                                  int64_t pitch)
{
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 8;
    if (c >= pitch) return;
    const T *X = blockIdx.z ? X1 : X0;
    T *out = blockIdx.z ? out1 : out0;
    const int64_t R = blockIdx.z ? R1 : R0;
    const int64_t step = static_cast<int64_t>(gridDim.y) * blockDim.y;
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; r < R; r += step) {
        float v[8];
        load8(X + r * C + c, C - c, v);
        store8(out + r * pitch + c, pitch - c, v);
    }
}

// dH [T][pitch] (zeros behind the N values) from dY [T, ncols] and the kept H; sums: per row chunk (blockIdx.y)
// the column sums [chunks][N] in fp32, before dH is rounded.  A block takes 512 columns (a wave 8 per lane) and
// every fourth row per wave.  Memory bound: SwiGLU over [4096, 2 x 14336] bfloat16 moves 704 MB and takes 135 us (the
// reads alone, for the sums, 75 us at 6.2 TB/s).  H, which nothing reads again, goes past the caches: 150 us without
// that; dY, which the step before has just written, does not (10 us more if it does).  Four waves side by side in one row
// instead of in four rows: 150 us.
constexpr int kSlopeCols = 512, kSlopeWaves = 4;
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void slope_kernel(const T *__restrict__ dY, const void *__restrict__ H, int64_t Ttok,
                                                    int64_t N, int64_t ncols, int64_t pitch, int64_t rows_per_chunk,
                                                    int act, T *__restrict__ dH, float *__restrict__ sums)
{
    __shared__ float s_sum[kSlopeWaves][GATED ? 2 : 1][kSlopeCols];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t left = ncols - (static_cast<int64_t>(blockIdx.x) * kSlopeCols + lane * 8);
    // the last columns of a row that is no multiple of 8: eight columns that end there, of which `again` are the
    // lane before's (the same values twice; they count once in the sums)
    const int again = left > 0 && left < 8 && ncols >= 8 ? 8 - static_cast<int>(left) : 0;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * kSlopeCols + lane * 8 - again;
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * rows_per_chunk;
    const int64_t r1 = r0 + rows_per_chunk < Ttok ? r0 + rows_per_chunk : Ttok;
    float sum[2][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[0][j] = sum[1][j] = 0.0f;
    // `here` columns exist: 8 as a constant where the loads need no cases and go out together
    auto rows = [&](auto here) {
#pragma unroll 2
        for (int64_t r = r0 + wave; r < r1; r += kSlopeWaves) {
            float d[8], h[8];
            load8(dY + r * ncols + c, here, d);
            if (GATED) {
                float a[8], g[8];
                kept8<T>(H, Ttok * N, r * N + c, here, a);
                kept8<T>(H, Ttok * N, r * N + ncols + c, here, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float s = logistic_for<T>(a[j]);
                    // (the factors of d are finite where a and g are; d a and d g alone may overflow where s is 0)
                    h[j] = d[j] * (a[j] * s);                                          // of the second half
                    d[j] = d[j] * (g[j] * (s + a[j] * s * (1.0f - s)));
                    sum[0][j] += d[j];
                    sum[1][j] += h[j];
                }
                if (dH) store8(dH + r * pitch + ncols + c, here, h);
            } else {
                if (act != OPMX_ACTIVATION_NONE) {
                    kept8<T>(H, Ttok * N, r * N + c, here, h);
#pragma unroll
                    for (int j = 0; j < 8; ++j) d[j] *= slope<T>(act, h[j]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[0][j] += d[j];
            }
            if (dH) {
                store8(dH + r * pitch + c, here, d);
                if (left <= 8)                                                         // the lane of the last columns
                    for (int64_t p = N; p < pitch; ++p) dH[r * pitch + p] = from_f32<T>(0.0f);
            }
        }
    };
    if (left >= 8 || again > 0) rows(std::integral_constant<int, 8>{});
    else if (left > 0) rows(left);
    if (sums == nullptr) return;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (j >= again) {
            s_sum[wave][0][lane * 8 + j - again] = sum[0][j];
            if (GATED) s_sum[wave][GATED ? 1 : 0][lane * 8 + j - again] = sum[1][j];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < kSlopeCols; i += 256) {
        const int64_t col = static_cast<int64_t>(blockIdx.x) * kSlopeCols + i;
        if (col >= ncols) break;
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (int v = 0; v < kSlopeWaves; ++v) {
            a += s_sum[v][0][i];
            if (GATED) b += s_sum[v][GATED ? 1 : 0][i];
        }
        sums[blockIdx.y * N + col] = a;
        if (GATED) sums[blockIdx.y * N + ncols + col] = b;
    }
}

// The chunks' column sums: a block takes 64 columns, each of its 16 waves every 16th chunk.
template <typename T>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float *__restrict__ sums, int64_t chunks, int64_t N,
                                                          T *__restrict__ dB)
{
    __shared__ double s_sum[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    double v = 0.0;
    if (c < N)
#pragma unroll 4
        for (int64_t i = wave; i < chunks; i += 16) v += sums[i * N + c];
    s_sum[wave][lane] = v;
    __syncthreads();
    if (wave == 0 && c < N) {
#pragma unroll
        for (int w = 1; w < 16; ++w) v += s_sum[w][lane];
        dB[c] = from_f32<T>(static_cast<float>(v));
    }
}

// The fp32 sums of the k ranges, added in order, through the epilogue.
constexpr int kJoin = 64;      // few values, long chains of loads: spread over as many CUs as there are
template <typename T, bool GATED>
__global__ __launch_bounds__(kJoin) void join_kernel(Epilogue e, int ranges)
{
    // (fewer than 2^31 values in ranges' sums of one range: see cut_for; a 64-bit division would cost a microsecond)
    const uint32_t chunks = static_cast<uint32_t>((e.ncols + 7) / 8), at = blockIdx.x * kJoin + threadIdx.x;
    const uint32_t row = at / chunks;
    if (row >= static_cast<uint64_t>(e.rows)) return;
    const int64_t m = row, c = static_cast<int64_t>(at - row * chunks) * 8;
    float h[8], g[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = g[j] = 0.0f;
    const float *p = e.part + m * e.pitch + c;
    const int64_t step = e.rows * e.pitch;
    int i = 0;
    for (; i + 4 <= ranges; i += 4, p += 4 * step) {          // four ranges' loads in flight
        float v[4][8], u[4][8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            load8(p + q * step, 8, v[q]);
            if (GATED) load8(p + q * step + e.pitch / 2, 8, u[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[j] += v[q][j];
                if (GATED) g[j] += u[q][j];
            }
    }
    for (; i < ranges; ++i, p += step) {
        float v[8];
        load8(p, 8, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += v[j];
        if (GATED) {
            load8(p + e.pitch / 2, 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] += v[j];
        }
    }
    const int64_t left = e.ncols - c;
    float bh[8], bg[8], res[8];
    load_bias8<T, GATED>(e, c, bh, bg);
    if (e.residual) load8(static_cast<const T *>(e.residual) + m * e.ncols + c, left, res);
    activate8<T, GATED>(e, m, c, left, bh, bg, h, g);
    if (e.residual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += res[j];
    }
    store8(static_cast<T *>(e.Y) + m * e.ncols + c, left, h);
}

// Tile and k ranges of a product of `rows` x `ncols` outputs (gated: ncols pairs of them) over Kc; p_rows, q_rows:
// k runs over the rows of P, of Q (Operand::k_major).
struct Cut {
    Tile tile;
    int ranges;
    int64_t pitch;      // of the ranges' sums
    size_t bytes;       // of the ranges' sums
};
// Of the tiles with less than 128 rows.
//
// Microseconds of a k-tile, of one workgroup on a CU and of two, and of joining r ranges, fitted to the times of 1 to 16
// ranges of 27 products with 20 to 3000 rows: the chosen ones are within 8 % of the best.  Returns the chosen one's.
double short_cut(Cut &c, int64_t rows, int64_t width, int64_t nk, bool p_rows, bool f32)
{
    const int64_t columns = ceil_div(width, 128);
    double best = 0;
    for (int half = 0; half < (f32 ? 2 : 1); ++half) {
        const double one = half ? 0.63 : f32 ? 1.1 : p_rows ? 0.45 : 0.34, two = half ? 1.25 : f32 ? 2.2 : p_rows ? 0.65 : 0.62;
        const int64_t tiles = ceil_div(rows, half ? 32 : 64) * columns;
        for (int64_t r = 1; r <= 16 && (r == 1 || r * 4 <= nk); ++r) {
            const int64_t load = ceil_div(tiles * r, 256);
            const double mb = static_cast<double>(r * rows * width) * 4e-6;
            const double us = static_cast<double>(ceil_div(nk, r)) *
                                  (static_cast<double>(load / 2) * two + static_cast<double>(load % 2) * one) +
                              (r > 1 ? 3.0 + 0.4 * static_cast<double>(r) + 0.3 * mb : 0.0);
            if ((half == 0 && r == 1) || us < best) {
                best = us;
                c.tile = half ? Tile::k32 : Tile::k64;
                c.ranges = static_cast<int>(r);
            }
        }
    }
    return best;
}
Cut cut_for(int64_t rows, int64_t ncols, int64_t Kc, bool gated, bool p_rows, bool q_rows, int dtype)
{
    Cut c{Tile::k128, 1, 0, 0};
    const bool f32 = dtype == OPMX_DTYPE_F32;
    const int64_t width = gated ? 2 * ncols : ncols, columns = ceil_div(width, 128);
    const int64_t nk = ceil_div(Kc, f32 ? 32 : 64);
    // The large tile needs most of the 256 CUs busy and k-tiles to spread its start and its end over: against 128 x 128,
    // 4096 x 8192 outputs over 16 k-tiles 76 us and 78, 4096 x 14336 over 4 77 and 57; with k over the rows of both
    // operands over 16 152 and 141, 4096 x 4096 over 32 66 and 75.  And rows for more than half of it: 64 x 49152 over 1024 31 and 20,
    // 128 x 65536 over 2048 64 and 53, 200 x 65536 over 2048 71 and 84.
    if (!f32 && rows > 128 && ceil_div(rows, 256) * ceil_div(width, 256) >= 192 && nk >= (q_rows ? 24 : 16)) {
        c.tile = Tile::k256;
        return c;
    }
    // More tiles than CUs: 128 x 128 (float16, 3000 x 2816 outputs over 2048: 54 us, 64 x 128 55, the gradients 47 and 55).
    // Fewer: 64 x 128 (512 x 1024 over 1024 9 us, 128 x 128 13; 100 x 2048 over 1408 11 and 17), with k in ranges where it is long.
    if (rows > 64 && ceil_div(rows, 128) * columns > 256) {
        // In fp32 the matrix units' time of the last round decides: microseconds of a k-tile, of one and of two workgroups on a CU.
        // 181 x 19264 over 1600 117 us in 64 x 128 tiles and 203 in 128 x 128, 3000 x 2816 over 2048 329 and 383, 8192 x 1024 over 1024
        // 149 and 130.  Over 1750 products of 65 to 28672 rows the chosen tile is 1.1 % over the best in the mean and 22 % at most.
        auto rounds = [](int64_t tiles, double one, double two) {
            const int64_t load = ceil_div(tiles, 256);
            return static_cast<double>(load / 2) * two + static_cast<double>(load % 2) * one;
        };
        if (f32 && rounds(ceil_div(rows, 64) * columns, 1.15, 2.2) < rounds(ceil_div(rows, 128) * columns, 1.93, 3.87)) c.tile = Tile::k64;
        return c;
    }
    // In fp32, where a tile of half the rows takes little more than half the matrix units' time, also 32 x 128 (512 x 1024
    // over 1024 18 us, 64 x 128 21; 2048 x 2048 over 2048 150, 135).
    short_cut(c, rows, width, nk, p_rows, f32);
    if (c.ranges > 1) c.ranges = static_cast<int>(ceil_div(nk, ceil_div(nk, c.ranges)));      // none of them empty
    if (c.ranges > 1) {
        c.pitch = gated ? 2 * up(ncols, 8) : up(ncols, 8);
        c.bytes = static_cast<size_t>(c.ranges) * rows * c.pitch * 4;
    }
    return c;
}

// Whether a forward pass goes without tiles (linear_few_rows.hip).  Both kinds of kernel are estimated; the tile product's time is
// that of its workgroups or of reading W, and rows that are not whole chunks are copied first.  Over the 3080 sizes
// the chosen one takes 0.6 % more than the quicker one in the mean, over 10 % at 85.  Microseconds here and in tiles: 1 x
// 4096 -> 4096 float16 8.2, 13.8; 20 x 1024 -> 4096 float16 5.4, 9.0; 32 x 4096 -> 1024 float16 14.5, 10.1; 64 x 1024 -> 2816 float32
// 13.0, 12.8; 64 x 1024 -> 28672 float16 43, 15; 16 x 4095 -> 4096 float32 27, 47; 16 x 14335 -> 1024 float16 88, 31.
bool few_rows_serve(int64_t Ttok, int64_t K, int64_t N, bool gated, int dtype)
{
    if (Ttok > 64) return false;
    const bool f32 = dtype == OPMX_DTYPE_F32;
    const int64_t size = f32 ? 4 : 2, width = gated ? 2 * (N / 2) : N;
    const double mb = static_cast<double>(N * K * size) * 1e-6;
    Cut c{};
    const double tiles = 3.7 + 0.9 * short_cut(c, Ttok, width, ceil_div(K, f32 ? 32 : 64), false, f32);
    const double copies = K * size % 16 == 0 ? 0.0 : 2.5 + mb / 2.4;
    return linear_few_rows_us(Ttok, K, N, dtype, gated) < std::max(tiles, 4.7 + mb / 4.7) + copies;
}

template <typename T> int join(const Epilogue &e, int ranges, hipStream_t s)
{
    const int64_t blocks = ceil_div(ceil_div(e.ncols, 8) * e.rows, kJoin);
    if (blocks >= (int64_t{1} << 25)) return OPMX_ERR_UNSUPPORTED;      // 32-bit counts in the kernel
    if (e.act == OPMX_ACTIVATION_SWIGLU) join_kernel<T, true><<<static_cast<unsigned>(blocks), kJoin, 0, s>>>(e, ranges);
    else join_kernel<T, false><<<static_cast<unsigned>(blocks), kJoin, 0, s>>>(e, ranges);
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

template <typename T>
int product(const Operand &P, const Operand &Q, int64_t Kc, Epilogue e, void *ws, hipStream_t s)
{
    const bool gated = e.act == OPMX_ACTIVATION_SWIGLU;
    const Cut c = cut_for(e.rows, e.ncols, Kc, gated, P.k_major, Q.k_major, DType<T>::id);
    if (c.ranges > 1) {
        e.part = static_cast<float *>(ws);
        e.pitch = c.pitch;
    }
    const int rc = launch_linear_gemm(P, Q, Kc, DType<T>::id, e, c.tile, c.ranges, s);
    return rc != OPMX_OK || c.ranges == 1 ? rc : join<T>(e, c.ranges, s);
}

struct Lanes {
    dim3 grid, block;
};
// 8 columns per lane, short rows several to a block.
inline Lanes lanes_over(int64_t rows, int64_t cols)
{
    int bx = 8;
    while (bx < 256 && bx * 8 < cols) bx <<= 1;
    const int64_t y = ceil_div(rows, 256 / bx);
    return {dim3(static_cast<unsigned>(ceil_div(cols, bx * 8)), static_cast<unsigned>(y < 65535 ? y : 65535)),
            dim3(bx, 256 / bx)};
}

template <typename T>
int pad(const void *X0, int64_t R0, void *out0, const void *X1, int64_t R1, void *out1, int64_t C, hipStream_t s)
{
    const int64_t pitch = up(C, 16 / sizeof(T));
    Lanes l = lanes_over(R0 > R1 ? R0 : R1, pitch);
    l.grid.z = X1 ? 2 : 1;
    pad_kernel<T><<<l.grid, l.block, 0, s>>>(static_cast<const T *>(X0), R0, static_cast<T *>(out0), static_cast<const T *>(X1),
                                             R1, static_cast<T *>(out1), C, pitch);
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

// What the workspace holds, in this order.
struct ForwardPlan {
    size_t x, w, part, total;
};
ForwardPlan forward_plan(int64_t Ttok, int64_t K, int64_t N, int dtype, int act)
{
    const int64_t esize = dtype == OPMX_DTYPE_F32 ? 4 : 2, n = 16 / esize, pitch = up(K, n);
    const bool gated = act == OPMX_ACTIVATION_SWIGLU, padded = K % n != 0;
    ForwardPlan p{};
    if (few_rows_serve(Ttok, K, N, gated, dtype)) return p;
    p.x = 0;
    p.w = p.x + (padded ? up(Ttok * pitch * esize, 256) : 0);
    p.part = p.w + (padded ? up(N * pitch * esize, 256) : 0);
    p.total = p.part + up(cut_for(Ttok, gated ? N / 2 : N, K, gated, false, false, dtype).bytes, 256);
    return p;
}

// Rows per chunk of the slope pass: 8 (two per wave) while that leaves at most 4096 blocks, then more; 512 chunks at most.
inline int64_t chunk_rows(int64_t Ttok, int64_t ncols)
{
    const int64_t strips = ceil_div(ncols, kSlopeCols);
    int64_t rows = 8;
    while ((ceil_div(Ttok, rows) * strips > 4096 && rows < 64) || ceil_div(Ttok, rows) > 512) rows <<= 1;
    return rows;
}

struct BackwardPlan {
    size_t dh, x, w, sums, part, total;
    int64_t pitch_n, pitch_k, chunk;
    bool own_dh, own_x, own_w;
};
// wanted: opmx_linear_gradient; only what these need has a place.
BackwardPlan backward_plan(int64_t Ttok, int64_t K, int64_t N, int dtype, int act, int wanted)
{
    const int64_t esize = dtype == OPMX_DTYPE_F32 ? 4 : 2, n = 16 / esize;
    const bool dX = wanted & OPMX_LINEAR_DX, dW = wanted & OPMX_LINEAR_DW, padded = K % n != 0;
    BackwardPlan p{};
    p.pitch_n = up(N, n);
    p.pitch_k = up(K, n);
    p.own_dh = (act != OPMX_ACTIVATION_NONE || N % n != 0) && (dX || dW);
    p.own_x = dW && (padded || (wanted & OPMX_LINEAR_X8));          // padded, or unpacked from 8 bits
    p.own_w = dX && padded;
    p.chunk = chunk_rows(Ttok, act == OPMX_ACTIVATION_SWIGLU ? N / 2 : N);
    p.dh = 0;
    p.x = p.dh + (p.own_dh ? up(Ttok * p.pitch_n * esize, 256) : 0);
    p.w = p.x + (p.own_x ? up(Ttok * p.pitch_k * esize, 256) : 0);
    p.sums = p.w + (p.own_w ? up(N * p.pitch_k * esize, 256) : 0);
    p.part = p.sums + (wanted & OPMX_LINEAR_DB ? up(ceil_div(Ttok, p.chunk) * N * 4, 256) : 0);
    const size_t a = dX ? cut_for(Ttok, K, N, false, true, false, dtype).bytes : 0;
    const size_t b = dW ? cut_for(N, K, Ttok, false, true, true, dtype).bytes : 0;
    p.total = p.part + up(a > b ? a : b, 256);
    return p;
}

template <typename T>
int forward_impl(const void *X, const void *W, const void *B, const void *R, int64_t Ttok, int64_t K, int64_t N, int act,
                 void *Y, void *H, char *ws, hipStream_t s)
{
    constexpr int64_t n = 16 / sizeof(T);
    Epilogue e;
    e.bias = B;
    e.residual = R;
    e.Y = Y;
    e.H = H;
    e.rows = Ttok;
    e.N = N;
    e.ncols = act == OPMX_ACTIVATION_SWIGLU ? N / 2 : N;
    e.act = act;
    if (few_rows_serve(Ttok, K, N, act == OPMX_ACTIVATION_SWIGLU, DType<T>::id)) return launch_linear_few_rows(X, W, K, DType<T>::id, e, s);
    const ForwardPlan plan = forward_plan(Ttok, K, N, DType<T>::id, act);
    int64_t pitch = K;
    if (K % n != 0) {
        pitch = up(K, n);
        const int rc = pad<T>(X, Ttok, ws + plan.x, W, N, ws + plan.w, K, s);
        if (rc != OPMX_OK) return rc;
        X = ws + plan.x;
        W = ws + plan.w;
    }
    return product<T>({W, pitch, false}, {X, pitch, false}, K, e, ws + plan.part, s);
}

template <typename T>
int backward_impl(const void *dY, const void *X, const void *xq, const void *xcode, const void *W, const void *H,
                  int64_t Ttok, int64_t K, int64_t N, int act, void *dX, void *dW, void *dB, int wanted, char *ws, hipStream_t s)
{
    const BackwardPlan plan = backward_plan(Ttok, K, N, DType<T>::id, act, wanted);
    const bool gated = act == OPMX_ACTIVATION_SWIGLU;
    const int64_t ncols = gated ? N / 2 : N;
    const void *dH = dY;
    int rc = OPMX_OK;
    if (Ttok > 0 && (plan.own_dh || dB)) {
        T *out = plan.own_dh ? reinterpret_cast<T *>(ws + plan.dh) : nullptr;
        float *sums = dB ? reinterpret_cast<float *>(ws + plan.sums) : nullptr;
        const dim3 grid(static_cast<unsigned>(ceil_div(ncols, kSlopeCols)), static_cast<unsigned>(ceil_div(Ttok, plan.chunk)));
        if (gated)
            slope_kernel<T, true><<<grid, 256, 0, s>>>(static_cast<const T *>(dY), H, Ttok, N, ncols,
                                                             plan.pitch_n, plan.chunk, act, out, sums);
        else
            slope_kernel<T, false><<<grid, 256, 0, s>>>(static_cast<const T *>(dY), H, Ttok, N, ncols,
                                                              plan.pitch_n, plan.chunk, act, out, sums);
        OPMX_LAUNCH_CHECK();
    }
    if (plan.own_dh) dH = ws + plan.dh;
    if (dB) {
        column_sum_kernel<T><<<static_cast<unsigned>(ceil_div(N, 64)), 1024, 0, s>>>(
            reinterpret_cast<const float *>(ws + plan.sums), ceil_div(Ttok, plan.chunk), N, static_cast<T *>(dB));
        OPMX_LAUNCH_CHECK();
    }
    // W and X as the products take them
    int64_t pitch_w = K, pitch_x = K;
    const bool pad_w = plan.own_w, pad_x = plan.own_x && !xq && Ttok > 0;
    if (pad_w && pad_x) rc = pad<T>(W, N, ws + plan.w, X, Ttok, ws + plan.x, K, s);
    else if (pad_w) rc = pad<T>(W, N, ws + plan.w, nullptr, 0, nullptr, K, s);
    else if (pad_x) rc = pad<T>(X, Ttok, ws + plan.x, nullptr, 0, nullptr, K, s);
    if (rc == OPMX_OK && dW && xq) rc = launch_checkpoint8_unpack(xq, xcode, Ttok, K, DType<T>::id, ws + plan.x, s, plan.pitch_k);
    if (rc != OPMX_OK) return rc;
    if (pad_w) {
        W = ws + plan.w;
        pitch_w = plan.pitch_k;
    }
    if (pad_x || (dW && xq)) {
        X = ws + plan.x;
        pitch_x = plan.pitch_k;
    }
    Epilogue e;
    if (dX) {
        e.Y = dX;
        e.rows = Ttok;
        e.N = e.ncols = K;
        rc = product<T>({W, pitch_w, true}, {dH, plan.pitch_n, false}, N, e, ws + plan.part, s);
        if (rc != OPMX_OK) return rc;
    }
    if (dW) {
        e.Y = dW;
        e.rows = N;
        e.N = e.ncols = K;
        rc = product<T>({X, pitch_x, true}, {dH, plan.pitch_n, true}, Ttok, e, ws + plan.part, s);
    }
    return rc;
}

}  // namespace

// 256 bytes say that none are needed, and that there may be no workspace: whatever is needed is more than that.
static size_t bytes_for(size_t total) { return total == 0 ? 256 : total < 512 ? 512 : total; }

size_t linear_epilogue_workspace_bytes(int64_t T, int64_t K, int64_t N, int dtype, int act)
{
    return bytes_for(forward_plan(T, K, N, dtype, act).total);
}
size_t linear_epilogue_backward_workspace_bytes(int64_t T, int64_t K, int64_t N, int dtype, int act, int wanted)
{
    return bytes_for(backward_plan(T, K, N, dtype, act, wanted).total);
}

int launch_linear_epilogue(const void *X, const void *W, const void *B, const void *R, int64_t T, int64_t K, int64_t N,
                           int dtype, int act, void *Y, void *H, void *ws, hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return forward_impl<float>(X, W, B, R, T, K, N, act, Y, H, static_cast<char *>(ws), s);
        case OPMX_DTYPE_F16: return forward_impl<f16>(X, W, B, R, T, K, N, act, Y, H, static_cast<char *>(ws), s);
        case OPMX_DTYPE_BF16: return forward_impl<bf16>(X, W, B, R, T, K, N, act, Y, H, static_cast<char *>(ws), s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

int launch_linear_epilogue_backward(const void *dY, const void *X, const void *xq, const void *xcode, const void *W,
                                    const void *H, int64_t T, int64_t K, int64_t N, int dtype, int act, void *dX, void *dW,
                                    void *dB, int wanted, void *ws, hipStream_t s)
{
    char *w = static_cast<char *>(ws);
    switch (dtype) {
        case OPMX_DTYPE_F32: return backward_impl<float>(dY, X, xq, xcode, W, H, T, K, N, act, dX, dW, dB, wanted, w, s);
        case OPMX_DTYPE_F16: return backward_impl<f16>(dY, X, xq, xcode, W, H, T, K, N, act, dX, dW, dB, wanted, w, s);
        case OPMX_DTYPE_BF16: return backward_impl<bf16>(dY, X, xq, xcode, W, H, T, K, N, act, dX, dW, dB, wanted, w, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

}  // namespace opmx
