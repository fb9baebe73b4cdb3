// Linear with epilogue for few rows of X (decoding: one token up to 32, 64 with short rows): reading W once at the memory's pace.
//
//   H[t, c] = sum_k X[t, k] W[c, k], then the epilogue
//
// A workgroup of eight waves owns 16 RT rows of W (with SwiGLU 16 of each half) and all rows of X over the whole of k:
// nothing has to be joined by a second launch.  The waves share out k in pieces of 128 bytes of a row and feed the
// MFMAs straight from global memory, one batch of pieces ahead; the partial sums meet in LDS and are added in wave
// order.  W is the A operand, so a lane holds four neighbouring columns of a row of Y.  X comes from L2: 16 RT rows
// of W share one reading of it, and a row of X past the last one is the last one again, never stored.
// Rows of W and X may start anywhere their type allows; the last k values that fill no piece go one by one.
#include "linear_epilogue.h"
#include "linear_step.h"

#include <algorithm>
#include <cmath>

namespace opmx {
namespace {

constexpr int kFewWaves = 8;
constexpr int64_t kFewWideColumns = 16384;       // from here on 32 columns per workgroup: 512 workgroups at least
constexpr int64_t kFewStreamBytes = 8 << 20;     // weights from which on they go through LDS

// 16 bytes at any address; `once`: what the caches need not keep.
template <typename F, bool ONCE> __device__ __forceinline__ F load_frag(const void *p)
{
    const quad_any q = ONCE ? __builtin_nontemporal_load(static_cast<const quad_any *>(p)) : *static_cast<const quad_any *>(p);
    F f;
    __builtin_memcpy(&f, &q, 16);
    return f;
}

// The end of both kernels: part holds the waves' sums [wave][tile of W][tile of X][lane].
template <typename T, int NT, int RT, bool GATED, int WAVES>
__device__ __forceinline__ void finish_rows(const float4_t (*part)[RT][NT][kWave], const Epilogue &e, int64_t c0)
{
    // a thread takes eight columns of a row: quads g = 2 c, 2 c + 1 of the row's lanes
    constexpr int CB = GATED ? 16 : 16 * RT, CHUNKS = CB / 8;
    for (int id = threadIdx.x; id < NT * 16 * CHUNKS; id += WAVES * kWave) {
        const int row = id / CHUNKS, chunk = id % CHUNKS;
        const int64_t c = c0 + chunk * 8, left = e.ncols - c;
        if (row >= e.rows || left <= 0) continue;
        float h[8], gate[8], bh[8], bg[8], res[8];
        load_bias8<T, GATED>(e, c, bh, bg);
        if (e.residual) load8(static_cast<const T *>(e.residual) + row * e.ncols + c, left, res);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int at = ((chunk % 2) * 2 + x) * 16 + row % 16;
            float4_t v{0.f, 0.f, 0.f, 0.f}, u = v;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                v += part[w][GATED ? 0 : chunk / 2][row / 16][at];
                if (GATED) u += part[w][RT - 1][row / 16][at];
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                h[x * 4 + y] = v[y];
                gate[x * 4 + y] = u[y];
            }
        }
        activate8<T, GATED>(e, row, c, left, bh, bg, h, gate);
        if (e.residual) {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] += res[j];
        }
        store8(static_cast<T *>(e.Y) + row * e.ncols + c, left, h);
    }
}

// NT: tiles of 16 rows of X; RT: tiles of 16 rows of W (GATED: 2, the second from the second half).
template <typename T, int NT, int RT, bool GATED>
__global__ __launch_bounds__(kFewWaves *kWave, 2) void few_rows_kernel(const T *__restrict__ X, const T *__restrict__ W, int64_t K,
                                                                        Epilogue e)
{
    using frag = typename Step<T>::frag;
    constexpr int n = 16 / sizeof(T), STEP = 4 * n;          // k values of a lane's load, of one MFMA step
    constexpr int U = NT * RT >= 4 ? 2 : 4;                  // steps of a batch; two batches are in flight
    constexpr int CB = GATED ? 16 : 16 * RT;                 // columns of Y per workgroup
    __shared__ __attribute__((aligned(16))) float4_t part[kFewWaves][RT][NT][kWave];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r = lane & 15, g = lane >> 4;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * CB;
    const T *wp[RT], *xp[NT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t c = c0 + (GATED ? 0 : i * 16) + r;
        const int64_t row = (c < e.ncols ? c : e.ncols - 1) + (GATED && i == 1 ? e.ncols : 0);
        wp[i] = W + row * K + g * n;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) xp[t] = X + (t * 16 + r < e.rows ? t * 16 + r : e.rows - 1) * K + g * n;
    float4_t acc[RT][NT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = float4_t{0.f, 0.f, 0.f, 0.f};

    // steps 2 v and 2 v + 1 (128 bytes of a row) belong to wave v mod 8; they go in batches of U, one batch's loads ahead
    const int steps = static_cast<int>(K / STEP);
    constexpr int AHEAD = U / 2 * 2 * kFewWaves;             // from a batch to the next
    int s = wave * 2;
    auto load = [&](int at, frag (&w)[U][RT], frag (&x)[U][NT]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = static_cast<int64_t>(at + u / 2 * 2 * kFewWaves + u % 2) * STEP;
#pragma unroll
            for (int i = 0; i < RT; ++i) w[u][i] = load_frag<frag, true>(wp[i] + k);
#pragma unroll
            for (int t = 0; t < NT; ++t) x[u][t] = load_frag<frag, false>(xp[t] + k);
        }
        __builtin_amdgcn_sched_barrier(0);                   // all of them before the next product
    };
    auto multiply = [&](const frag (&w)[U][RT], const frag (&x)[U][NT]) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = Step<T>::mma(w[u][i], x[u][t], acc[i][t]);
        __builtin_amdgcn_sched_barrier(0);
    };
    const int last = steps - ((U / 2 - 1) * 2 * kFewWaves + 2);       // where a whole batch may begin at most
    if (s <= last) {
        frag wa[U][RT], xa[U][NT], wb[U][RT], xb[U][NT];
        load(s, wa, xa);
        for (; s + 2 * AHEAD <= last; s += 2 * AHEAD) {
            load(s + AHEAD, wb, xb);
            multiply(wa, xa);
            load(s + 2 * AHEAD, wa, xa);
            multiply(wb, xb);
        }
        if (s + AHEAD <= last) {
            load(s + AHEAD, wb, xb);
            multiply(wa, xa);
            multiply(wb, xb);
            s += AHEAD;
        } else {
            multiply(wa, xa);
        }
        s += AHEAD;
    }
    for (; s < steps; s += 2 * kFewWaves)
        for (int u = 0; u < 2 && s + u < steps; ++u) {
            const int64_t k = static_cast<int64_t>(s + u) * STEP;
            frag w[RT], x[NT];
#pragma unroll
            for (int i = 0; i < RT; ++i) w[i] = load_frag<frag, true>(wp[i] + k);
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] = load_frag<frag, false>(xp[t] + k);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = Step<T>::mma(w[i], x[t], acc[i][t]);
        }
    if (K % STEP != 0 && wave == kFewWaves - 1) {            // the values behind the last whole step
        const int64_t k = static_cast<int64_t>(steps) * STEP, left = K - k - g * n;
        frag w[RT], x[NT];
        auto tail = [&](const T *p) {
            T v[n];
#pragma unroll
            for (int j = 0; j < n; ++j) v[j] = p[k + (j < left ? j : left - 1)];       // (p + k + left - 1: the row's last)
#pragma unroll
            for (int j = 0; j < n; ++j) v[j] = j < left ? v[j] : from_f32<T>(0.0f);
            frag f;
            __builtin_memcpy(&f, v, 16);
            return f;
        };
#pragma unroll
        for (int i = 0; i < RT; ++i) w[i] = tail(wp[i]);
#pragma unroll
        for (int t = 0; t < NT; ++t) x[t] = tail(xp[t]);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][t] = Step<T>::mma(w[i], x[t], acc[i][t]);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) part[wave][i][t][lane] = acc[i][t];
    __syncthreads();

    finish_rows<T, NT, RT, GATED, kFewWaves>(part, e, c0);
}

// ---------------------------------------------------------------------------------------------------------
// The same for more weights than a moment's reading: W comes through LDS in pieces of 16 RT rows x 512 bytes, so that memory
// sees that much of a row at a time, SLOTS - 1 pieces ahead.  The waves share a piece's k, two MFMA steps each.
// One token, weights not in any cache: 28672 x 4096 SwiGLU fp16 39 us = 6.0 TB/s (the kernel above 47, the tile product 50),
// 4096 x 4096 8.2 us (9.2, 13.8), 4096 x 14336 22.5 us (29, 27).
constexpr uint32_t kNowhere = 0x80000000u;      // past every descriptor
constexpr int kNonTemporal = 2;

// 16 bytes per lane from base + off to lds + 16 * lane; what lies past the descriptor reads as zero.
template <int POLICY> __device__ __forceinline__ void rows_to_lds(const char *base, char *lds, uint32_t off)
{
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b >> 32));
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
        reinterpret_cast<void *>((static_cast<uint64_t>(hi) << 32) | lo), 0, 0x7FFFFFFF, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, OPMX_LDS(lds), 16, off, 0, 0, POLICY);
}
// Until at most N of the wave's loads are outstanding (they land in order) and all its LDS reads are done.
template <int N> __device__ __forceinline__ void wait_few()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

template <typename T, int NT, int RT, int WAVES, int SLOTS, bool GATED>
__global__ __launch_bounds__(WAVES *kWave) void few_rows_stream_kernel(const T *__restrict__ X, const T *__restrict__ W, int64_t K,
                                                              Epilogue e)
{
    using frag = typename Step<T>::frag;
    constexpr int PIECE = WAVES * 128, n = 16 / sizeof(T), BK = PIECE / sizeof(T);      // two MFMA steps per wave
    constexpr int CB = GATED ? 16 : 16 * RT, LOADS = 2 * (RT + NT), SLOT = 16 * (RT + NT) * PIECE;
    constexpr int PER_LOAD = 1024 / PIECE, LANES = kWave / PER_LOAD;                   // rows of a wave's load, lanes of a row
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r = lane & 15, g = lane >> 4;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * CB, bytes = K * sizeof(T);
    const char *wbase = reinterpret_cast<const char *>(W + c0 * K), *xbase = reinterpret_cast<const char *>(X);
    const char *wsecond = GATED ? wbase + e.ncols * bytes : wbase;

    // load i of the wave: one or two rows' pieces, 16-byte chunk c of row R in place c ^ (R mod 16)
    uint32_t off[LOADS];
    int first_k[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int row = (i * WAVES + wave) * PER_LOAD + lane / LANES, chunk = (lane % LANES) ^ (row & 15);
        first_k[i] = chunk * n;
        int64_t of;
        bool there;
        if (i < 2 * RT) {                       // W
            of = GATED ? row % 16 : row;
            there = c0 + of < e.ncols;
        } else {
            of = row - 16 * RT;
            there = of < e.rows;
        }
        off[i] = there ? static_cast<uint32_t>(of * bytes + chunk * 16) : kNowhere;
    }
    const int pieces = static_cast<int>((K + BK - 1) / BK);
    int64_t k_left = K;
    int fill = 0;
    auto load_next = [&]() {
        const int left = k_left < BK ? static_cast<int>(k_left) : BK;
        char *slot = smem + fill * SLOT;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const uint32_t v = first_k[i] < left ? off[i] : kNowhere;
            char *to = slot + (i * WAVES + wave) * 1024;
            if (i < 2 * RT) rows_to_lds<kNonTemporal>(GATED && i >= 2 ? wsecond : wbase, to, v);
            else rows_to_lds<0>(xbase, to, v);
        }
        wbase += PIECE;
        wsecond += PIECE;
        xbase += PIECE;
        k_left -= BK;
        fill = fill + 1 == SLOTS ? 0 : fill + 1;
    };
    float4_t acc[RT][NT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SLOTS - 1; ++i) load_next();
    int use = 0;
    for (int p = 0; p < pieces; ++p) {
        // this wave's loads of piece p have landed, its reads of piece p - 1 are done; then the others'
        wait_few<(SLOTS - 2) * LOADS>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        load_next();                            // where piece p - 1 was; past the end from nowhere
        const char *slot = smem + use * SLOT;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int place = (((wave * 2 + u) * 4 + g) ^ r) << 4;
            frag w[RT], x[NT];
#pragma unroll
            for (int i = 0; i < RT; ++i) w[i] = *reinterpret_cast<const frag *>(slot + (i * 16 + r) * PIECE + place);
#pragma unroll
            for (int t = 0; t < NT; ++t) x[t] = *reinterpret_cast<const frag *>(slot + ((RT + t) * 16 + r) * PIECE + place);
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[i][t] = Step<T>::mma(w[i], x[t], acc[i][t]);
        }
        use = use + 1 == SLOTS ? 0 : use + 1;
    }
    wait_few<0>();                              // the sums use the same memory
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    float4_t(*part)[RT][NT][kWave] = reinterpret_cast<float4_t(*)[RT][NT][kWave]>(smem);
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) part[wave][i][t][lane] = acc[i][t];
    __syncthreads();
    finish_rows<T, NT, RT, GATED, WAVES>(part, e, c0);
}

template <typename T, int NT, int RT, int WAVES, int SLOTS, bool GATED>
int few_rows_stream(const void *X, const void *W, int64_t K, const Epilogue &e, hipStream_t s)
{
    constexpr int SMEM = SLOTS * 16 * (RT + NT) * WAVES * 128, CB = GATED ? 16 : 16 * RT;
    static_assert(SMEM <= 160 * 1024 && SMEM >= WAVES * RT * NT * kWave * 16, "LDS, also for the sums");
    static_assert((SLOTS - 2) * 2 * (RT + NT) < 64, "six bits of counter");
    static std::atomic<uint64_t> done{0};
    const void *k = reinterpret_cast<const void *>(&few_rows_stream_kernel<T, NT, RT, WAVES, SLOTS, GATED>);
    if (!ensure_dynamic_smem(k, SMEM, done)) return OPMX_ERR_LAUNCH;
    few_rows_stream_kernel<T, NT, RT, WAVES, SLOTS, GATED><<<static_cast<unsigned>(ceil_div(e.ncols, CB)), WAVES * kWave, SMEM, s>>>(
        static_cast<const T *>(X), static_cast<const T *>(W), K, e);
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

template <typename T, int NT> int few_rows(const void *X, const void *W, int64_t K, const Epilogue &e, hipStream_t s)
{
    const T *x = static_cast<const T *>(X), *w = static_cast<const T *>(W);
    const unsigned grid = static_cast<unsigned>(ceil_div(e.ncols, 16));
    if (e.act == OPMX_ACTIVATION_SWIGLU) few_rows_kernel<T, NT, 2, true><<<grid, kFewWaves * kWave, 0, s>>>(x, w, K, e);
    else few_rows_kernel<T, NT, 1, false><<<grid, kFewWaves * kWave, 0, s>>>(x, w, K, e);
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

// Through LDS from kFewStreamBytes of weights on, with at most 16 rows of X: pieces of 512 bytes and two workgroups
// per CU.  1024 bytes by eight waves, deeper pieces, and workgroups that start k apart were not faster.
template <typename T> int few_rows_by_size(const void *X, const void *W, int64_t K, const Epilogue &e, hipStream_t s)
{
    if (e.rows > 32) return few_rows<T, 4>(X, W, K, e, s);
    if (e.rows > 16) return few_rows<T, 2>(X, W, K, e, s);
    const bool whole = K * sizeof(T) % 16 == 0 && aligned16(X) && aligned16(W);
    if (!whole || e.N * K * static_cast<int64_t>(sizeof(T)) < kFewStreamBytes) return few_rows<T, 1>(X, W, K, e, s);
    if (e.act == OPMX_ACTIVATION_SWIGLU) return few_rows_stream<T, 1, 2, 4, 3, true>(X, W, K, e, s);
    if (e.ncols >= kFewWideColumns) return few_rows_stream<T, 1, 2, 4, 3, false>(X, W, K, e, s);
    return few_rows_stream<T, 1, 1, 4, 5, false>(X, W, K, e, s);
}

}  // namespace

// Fitted, as the tile product's time in linear_epilogue.hip, to both kernels' times at 3080 sizes (1 to 64 rows, K 255 to 14336,
// N 128 to 28672, float16 and float32, plain and gated, K whole chunks and not, weights out of any cache; bfloat16 is
// float16): within 15 %, mostly.  A workgroup's time goes with the bytes of a row (kb) and the tiles of W and of X that it
// multiplies, and the CUs take them in rounds; through LDS it is that or the memory's pace.
double linear_few_rows_us(int64_t T, int64_t K, int64_t N, int dtype, bool gated)
{
    const int64_t size = dtype == OPMX_DTYPE_F32 ? 4 : 2, ncols = gated ? N / 2 : N;
    const double kb = static_cast<double>(K * size) / 1024, mb = static_cast<double>(N * K * size) * 1e-6;
    const bool whole = K * size % 16 == 0;
    const int tiles_w = gated ? 2 : 1, tiles_x = T <= 16 ? 1 : T <= 32 ? 2 : 4;
    const double workgroups = static_cast<double>(ceil_div(ncols, 16));
    if (T <= 16 && whole && N * K * size >= kFewStreamBytes) {
        const bool wide = !gated && ncols >= kFewWideColumns;
        const double us = 3.0 + std::ceil((wide ? workgroups / 2 : workgroups) / 512) * kb * (0.36 * (wide ? 2 : tiles_w) + 0.15);
        return std::max(us, 3.9 + mb / 5.75);
    }
    // rows that start anywhere: 16-byte loads across cache lines, more of them in the 16-bit types
    const double odd = whole ? 0.0 : size == 2 ? 1.1 * tiles_w - 0.35 * tiles_x + 1.5 * static_cast<double>(T) / 16 : 0.45;
    const double us = 2.0 + std::ceil(workgroups / 256) * (1.1 + kb * (0.55 * tiles_w + 0.45 * tiles_x + odd));
    return std::max(us, mb / 3.3);
}

int launch_linear_few_rows(const void *X, const void *W, int64_t K, int dtype, const Epilogue &e, hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return few_rows_by_size<float>(X, W, K, e, s);
        case OPMX_DTYPE_F16: return few_rows_by_size<f16>(X, W, K, e, s);
        case OPMX_DTYPE_BF16: return few_rows_by_size<bf16>(X, W, K, e, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

}  // namespace opmx
