// Tile product of the linear with epilogue, for the forward pass and both gradients (gfx950, MFMA).
//
//   C[m, c] = sum_k Q(m, k) P(c, k)
//     forward      Q = X  [T,K],  P = W [N,K]:  rows of both run along k
//     gradient X   Q = dH [T,N],  P = W [N,K] read as (c = K, k = N): k runs over rows
//     gradient W   Q = dH [T,N],  P = X [T,K], k = T: k runs over rows in both
//
// A workgroup owns a BM x BN tile of C and walks k in tiles of 128 bytes (64 values, 32 in fp32), loaded straight into
// LDS and one or two tiles ahead.  P is the A operand of the MFMAs and Q the B operand, so a lane ends up with four
// neighbouring columns of a row.
//   rows along k:     LDS [row][8 chunks of 16 bytes], chunk c in slot c ^ (row / 2 % 8): a fragment is one
//                     16-byte read, conflict free;
//   k along rows:     LDS [k][row], 16-bit fragments through the transposing LDS read (four k of one column per
//                     lane and read), fp32 ones value by value.  32-byte units (fp32: 64) are permuted within
//                     256 bytes by k so that the k rows that one read meets lie in different banks.
// What does not exist (rows, columns, k past the end) is loaded from an offset that the descriptor's range check
// answers with zeros.  The k order of a fragment is the same in both layouts, whatever it is.
#include "linear_epilogue.h"
#include "linear_step.h"

#include <type_traits>

namespace opmx {
namespace {

constexpr int kTileBytes = 128;                 // of k per row
constexpr uint32_t kNowhere = 0x80000000u;      // past every descriptor

__device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor(const char *base)
{
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(b >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>((static_cast<uint64_t>(hi) << 32) | lo), 0,
                                             0x7FFFFFFF, 0x00020000);
}

// How k-major rows are permuted inside a k row of LDS (ROWS values): the index of a unit (32 bytes; fp32: 64) is xored with
// this.  A transposing read takes, for every half of the wave, one unit of k rows 0 to 3 and 8 to 11 (from a multiple of
// 16): with 256 bytes per k row and more these differ in all three bits, with 128 bytes the parity of k already tells the
// halves of the banks apart.
template <typename T, int ROWS> __device__ __forceinline__ int unit_swizzle(int k)
{
    if constexpr (sizeof(T) == 4) return (k >> 2) & (ROWS >= 64 ? 3 : 1);      // as many units as a k row has, four at most
    else if constexpr (ROWS * sizeof(T) >= 256) return (k & 3) | ((k >> 3 & 1) << 2);
    else return (k >> 1 & 1) | ((k >> 3 & 1) << 1);
}

// Waits until at most N of the wave's loads are outstanding (they land in order) and all its LDS reads are done.
template <int N> __device__ __forceinline__ void wait_loads()
{
    static_assert(N < 64, "the counter has six bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// One operand's share of a thread: LOADS 16-byte pieces of a k-tile of ROWS rows.
template <typename T, int ROWS, int THREADS, bool KM, bool GATED> struct Loader {
    static constexpr int n = 16 / sizeof(T);
    static constexpr int LOADS = ROWS * kTileBytes / 16 / THREADS;
    const char *base, *base2;        // of the current k-tile (GATED: of the second half's rows)
    int64_t step;                    // to the next one
    uint32_t off[LOADS];
    int first_k[LOADS];              // within the tile

    // Rows [row0, row0 + ROWS) of `count`.  GATED: groups of 64 tile rows are 32 rows of the first half and the 32
    // rows of the second half (count further on) that belong to the same columns.
    __device__ __forceinline__ void init(const Operand &o, int64_t row0, int64_t count, int64_t k0)
    {
        const int64_t esize = sizeof(T);
        const char *p = static_cast<const char *>(o.p);
        if (KM) {
            base = p + (k0 * o.pitch + row0) * esize;
            base2 = base;
            step = (kTileBytes / sizeof(T)) * o.pitch * esize;
        } else {
            base = p + (row0 * o.pitch + k0) * esize;
            base2 = GATED ? base + count * o.pitch * esize : base;
            step = kTileBytes;
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int piece = i * THREADS + threadIdx.x;
            if (KM) {
                constexpr int per_k = ROWS / n;                  // pieces of a k row
                constexpr int per_unit = sizeof(T) == 2 ? 2 : 4;
                const int k = piece / per_k, c = piece % per_k;
                const int r = (((c / per_unit) ^ unit_swizzle<T, ROWS>(k)) * per_unit + c % per_unit) * n;
                first_k[i] = k;
                off[i] = row0 + r < count ? static_cast<uint32_t>((k * o.pitch + r) * esize) : kNowhere;
            } else {
                const int row = piece >> 3, c = (piece & 7) ^ ((row >> 1) & 7);
                const int r = GATED ? (row / 64) * 32 + row % 32 : row;
                first_k[i] = c * n;
                off[i] = row0 + r < count ? static_cast<uint32_t>(r * o.pitch * esize + c * 16) : kNowhere;
            }
        }
    }
    // Loads piece i of the current k-tile, of which k_left values exist, to lds + its place.
    __device__ __forceinline__ void issue(int i, char *lds, int k_left) const
    {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        const int piece0 = i * THREADS + wave * kWave;                       // of the wave: uniform
        const bool second = GATED && !KM && ((piece0 >> 3) % 64) >= 32;
        const uint32_t v = first_k[i] < k_left ? off[i] : kNowhere;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(descriptor(second ? base2 : base), OPMX_LDS(lds + piece0 * 16), 16, v, 0, 0, 0);
    }
    __device__ __forceinline__ void next()
    {
        base += step;
        base2 += step;
    }
};

// Transposing reads, waited for: the fragments of four (two) groups of 16 rows of a k-major tile.  One block of assembly
// because the compiler puts a wait for every outstanding global -> LDS load in front of the builtin (it takes it for a
// store), and the next k-tiles' loads are in flight by design.  a: LDS addresses of the fragments' lanes at k step 0.
typedef uint32_t u32pair __attribute__((ext_vector_type(2)));
template <int KSTEP_BYTES, int HALF_BYTES, typename F>
__device__ __forceinline__ void transposed4(F *f, const uint32_t *a)
{
    u32pair v[8];
    asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(KSTEP_BYTES), "n"(KSTEP_BYTES + HALF_BYTES)
                 : "memory");
#pragma unroll
    for (int j = 0; j < 4; ++j) __builtin_memcpy(&f[j], &v[2 * j], 16);
}
template <int KSTEP_BYTES, int HALF_BYTES, typename F>
__device__ __forceinline__ void transposed2(F *f, const uint32_t *a)
{
    u32pair v[4];
    asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\t"
                 "ds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
                 "ds_read_b64_tr_b16 %2, %5 offset:%6\n\t"
                 "ds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                 : "v"(a[0]), "v"(a[1]), "n"(KSTEP_BYTES), "n"(KSTEP_BYTES + HALF_BYTES)
                 : "memory");
#pragma unroll
    for (int j = 0; j < 2; ++j) __builtin_memcpy(&f[j], &v[2 * j], 16);
}

// The fragments of N groups of 16 rows from row 16 * row16 on, k step KS (0, 1), of an LDS tile of ROWS rows.
template <typename T, int ROWS, bool KM, int KS, int N>
__device__ __forceinline__ void fragments(const char *lds, int row16, int lane, typename Step<T>::frag (&f)[N])
{
    using frag = typename Step<T>::frag;
    const int r = lane & 15, g = lane >> 4;
    if constexpr (!KM) {
        const int slot = (KS * 4 + g) ^ ((r >> 1) & 7);
#pragma unroll
        for (int i = 0; i < N; ++i)
            f[i] = *reinterpret_cast<const frag *>(lds + ((row16 + i) * 16 + r) * kTileBytes + slot * 16);
    } else if constexpr (sizeof(T) == 2) {
        // lane r of a group of 16 reads four columns of k row r / 4 and receives four k rows of column r
        static_assert(N % 4 == 0 || N == 2, "four or two fragments per block of reads");
        constexpr int B = N < 4 ? 2 : 4;
        const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(OPMX_LDS(lds)));
        const int k = g * 8 + (r >> 2);             // neither the second half (k + 4) nor KS (k + 32) changes the swizzle
#pragma unroll
        for (int i = 0; i < N; i += B) {
            uint32_t a[B];
#pragma unroll
            for (int j = 0; j < B; ++j)
                a[j] = base + k * (ROWS * 2) + (((row16 + i + j) ^ unit_swizzle<T, ROWS>(k)) << 5) + (r & 3) * 8;
            if constexpr (B == 4) transposed4<KS * 32 * ROWS * 2, 4 * ROWS * 2>(f + i, a);
            else transposed2<KS * 32 * ROWS * 2, 4 * ROWS * 2>(f + i, a);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = KS * 16 + g * 4 + j;
                f[i][j] = *reinterpret_cast<const float *>(lds + k * (ROWS * 4) + (((row16 + i) ^ unit_swizzle<T, ROWS>(k)) << 6) + r * 4);
            }
    }
}

// Tile ids to tiles.  Ids go round the 8 XCDs; each XCD takes a contiguous eighth of the tiles, in bands of 8
// row tiles walked column by column, so that the 32 workgroups an XCD runs share 8 + 4 operand tiles in its L2.
// (32-bit throughout: a launch has fewer than 2^31 tiles, and a 64-bit division takes microseconds of a lone wave.)
__device__ __forceinline__ void place(uint32_t id, uint32_t mt, uint32_t nt, int64_t &m, int64_t &c)
{
    const uint32_t total = mt * nt, per = total / 8, rest = total % 8, x = id % 8;
    const uint32_t t = x * per + (x < rest ? x : rest) + id / 8;
    const uint32_t band = t / (8 * nt), first = band * 8;
    const uint32_t high = mt - first < 8 ? mt - first : 8;
    const uint32_t in = t - band * 8 * nt, col = in / high;
    m = first + (in - col * high);
    c = col;
}

// What becomes of a wave's tile: acc[j][i] holds row 16 i + lane % 16 and columns 16 j + 4 (lane / 16) + v.  It goes through
// LDS in pieces of (up to) 64 x 64 fp32 values of the wave's own (16-byte chunks xored with the row), so that a lane
// then has eight neighbouring columns of a row.  m0, c0: the first row and (output) column.
template <typename T, int TM, int TN, bool GATED>
__device__ __forceinline__ void write_columns(const float4_t (&acc)[TN][TM], const Epilogue &e, int64_t m0, int64_t c0, int lane,
                                              char *mine)
{
    constexpr int PIECE = TM < 4 ? TM * 16 : 64, DOWN = TM * 16 / PIECE, PIECES = DOWN * (TN / 4);
    const int r = lane & 15, g = lane >> 4;
    constexpr int PER_ROW = GATED ? 4 : 8, ROWS = kWave / PER_ROW;       // lanes per row, rows per trip
    const int c8 = lane % PER_ROW;
    auto staged = [&](int row, int chunk) { return reinterpret_cast<float4_t *>(mine + row * 256 + ((chunk ^ (row & 15)) << 4)); };
#pragma unroll 1
    for (int p = 0; p < PIECES; ++p) {                   // (the code behind the staging stands once)
        const int piece = p % DOWN;
        const int64_t c = c0 + p / DOWN * (GATED ? 32 : 64) + c8 * 8, left = e.ncols - c;
        float bias_h[8], bias_g[8];
        load_bias8<T, GATED>(e, c, bias_h, bias_g);
#pragma unroll
        for (int u = 0; u < PIECES; ++u)
            if (p == u) {
#pragma unroll
                for (int i = 0; i < PIECE / 16; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *staged(i * 16 + r, j * 4 + g) = acc[u / DOWN * 4 + j][u % DOWN * (PIECE / 16) + i];
            }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
        if (e.part) {
#pragma unroll 2
            for (int t = 0; t < PIECE / ROWS; ++t) {
                const int row = t * ROWS + lane / PER_ROW;
                const int64_t m = m0 + piece * PIECE + row;
                if (m >= e.rows || left <= 0) continue;
                float *at = e.part + (blockIdx.y * e.rows + m) * e.pitch + c;      // whole chunks: the pitch holds them
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    *reinterpret_cast<float4_any *>(at + x * 4) = *staged(row, c8 * 2 + x);
                    if (GATED) *reinterpret_cast<float4_any *>(at + e.pitch / 2 + x * 4) = *staged(row, 8 + c8 * 2 + x);
                }
            }
        } else {
            const bool shaped = GATED || e.act != OPMX_ACTIVATION_NONE || e.H;
            constexpr int GROUP = PIECE / ROWS < 4 ? PIECE / ROWS : 4;              // residual rows in flight
#pragma unroll 1
            for (int t0 = 0; t0 < PIECE / ROWS; t0 += GROUP) {
                float res[GROUP][8];
#pragma unroll
                for (int t = 0; t < GROUP; ++t) {
                    const int64_t m = m0 + piece * PIECE + (t0 + t) * ROWS + lane / PER_ROW;
                    if (e.residual && m < e.rows && left > 0)
                        load8(static_cast<const T *>(e.residual) + m * e.ncols + c, left, res[t]);
                }
                if (shaped) {
                    // in place, in a rolled loop: the code of eight activations once
#pragma unroll 1
                    for (int t = t0; t < t0 + GROUP; ++t) {
                        const int row = t * ROWS + lane / PER_ROW;
                        const int64_t m = m0 + piece * PIECE + row;
                        if (m >= e.rows || left <= 0) continue;
                        float h[8], gate[8];
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float4_t v = *staged(row, c8 * 2 + x);
                            const float4_t u = GATED ? *staged(row, 8 + c8 * 2 + x) : v;
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                h[x * 4 + y] = v[y];
                                gate[x * 4 + y] = u[y];
                            }
                        }
                        activate8<T, GATED>(e, m, c, left, bias_h, bias_g, h, gate);
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            *staged(row, c8 * 2 + x) = float4_t{h[x * 4], h[x * 4 + 1], h[x * 4 + 2], h[x * 4 + 3]};
                    }
                }
#pragma unroll
                for (int t = 0; t < GROUP; ++t) {
                    const int row = (t0 + t) * ROWS + lane / PER_ROW;
                    const int64_t m = m0 + piece * PIECE + row;
                    if (m >= e.rows || left <= 0) continue;
                    float h[8];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float4_t v = *staged(row, c8 * 2 + x);
#pragma unroll
                        for (int y = 0; y < 4; ++y) h[x * 4 + y] = v[y];
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] += (shaped ? 0.0f : bias_h[j]) + (e.residual ? res[t][j] : 0.0f);
                    store8(static_cast<T *>(e.Y) + m * e.ncols + c, left, h);
                }
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool PK, bool QK, bool GATED>
__global__ __launch_bounds__(WM *WN *kWave, 2) void linear_gemm_kernel(Operand P, Operand Q, int64_t Kc, Epilogue e, uint32_t mt,
                                                                    uint32_t nt, int64_t ktiles_per_range)
{
    constexpr int THREADS = WM * WN * kWave, WTM = BM / WM, WTN = BN / WN, TM = WTM / 16, TN = WTN / 16;
    constexpr int STAGE = (BM + BN) * kTileBytes, BK = kTileBytes / sizeof(T);
    constexpr int BNO = GATED ? BN / 2 : BN;
    constexpr int PIECE = WTM < 64 ? WTM : 64;
    static_assert(WTN == 64 && (TM == 1 || TM == 2 || TM == 4), "the epilogue stages pieces of 64 columns");
    using frag = typename Step<T>::frag;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    int64_t tm, tc;
    place(blockIdx.x, mt, nt, tm, tc);
    const int64_t m0 = tm * BM, c0 = tc * BNO;
    const int64_t kt0 = blockIdx.y * ktiles_per_range;
    const int64_t k0 = kt0 * BK;
    const int64_t klen = Kc - k0 < ktiles_per_range * BK ? Kc - k0 : ktiles_per_range * BK;   // > 0: see the launch
    const int nk = static_cast<int>((klen + BK - 1) / BK);
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave / WN, wn = wave % WN;

    Loader<T, BN, THREADS, PK, GATED> lp;
    Loader<T, BM, THREADS, QK, false> lq;
    lp.init(P, c0, e.ncols, k0);
    lq.init(Q, m0, e.rows, k0);

    float4_t acc[TN][TM];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[j][i] = float4_t{0.f, 0.f, 0.f, 0.f};

    auto load = [&](char *stage, int64_t k_left) {
        const int left = k_left < BK ? static_cast<int>(k_left) : BK;
#pragma unroll
        for (int i = 0; i < lq.LOADS; ++i) lq.issue(i, stage, left);
#pragma unroll
        for (int i = 0; i < lp.LOADS; ++i) lp.issue(i, stage + BM * kTileBytes, left);
        lq.next();
        lp.next();
    };
    auto multiply = [&](const char *cur, auto ks_tag) {
        constexpr int KS = decltype(ks_tag)::value;
        frag p[TN], q[TM];
        fragments<T, BN, PK, KS, TN>(cur + BM * kTileBytes, wn * TN, lane, p);
        fragments<T, BM, QK, KS, TM>(cur, wm * TM, lane, q);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[j][i] = Step<T>::mma(p[j], q[i], acc[j][i]);
    };
    // STAGES - 1 k-tiles are on their way at any time.  Past the last one the loads go on, from nowhere, so that the
    // number of outstanding ones that means "tile kt has landed" stays the same.
    constexpr int AHEAD = (STAGES - 2) * (decltype(lp)::LOADS + decltype(lq)::LOADS);
    int64_t k_left = klen;
    int fill = 0;                                          // the stage that the next tile goes to
    auto load_next = [&]() {
        load(smem + fill * STAGE, k_left);
        k_left -= BK;
        fill = fill + 1 == STAGES ? 0 : fill + 1;
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) load_next();
    int stage = 0;
    for (int kt = 0; kt < nk; ++kt) {
        wait_loads<AHEAD>();                               // this wave's loads of tile kt, and its reads of tile kt - 1
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char *cur = smem + stage * STAGE;
        // Into the stage that tile kt - 1 was in, when the first products are under way (512 x 1024 over 1024 bfloat16 9.0 us, ahead of
        // them 9.5; 3000 x 2816 over 2048 float32 365, 378; gradient of X 2048 x 4096 over 14336 bfloat16 208, 223); with two stages
        // in LDS and the quickest products every moment counts for the loads (3000 x 2816 over 2048 bfloat16 54, ahead 51).
        constexpr bool ahead = STAGES == 2 && sizeof(T) == 2 && !PK;
        if constexpr (ahead) load_next();
        multiply(cur, std::integral_constant<int, 0>{});
        if constexpr (!ahead) load_next();
        multiply(cur, std::integral_constant<int, 1>{});
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    wait_loads<0>();                                       // the epilogue uses the same memory
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    write_columns<T, TM, TN, GATED>(acc, e, m0 + wm * WTM, c0 + wn * (GATED ? 32 : 64), lane, smem + wave * (PIECE * 256));
}

// ---------------------------------------------------------------------------------------------------------
// The product of many rows (16-bit types): 256 x 256 tiles, four waves of 128 x 128.
//
// Against eight waves of 128 x 64 the wave tiles read a third less from LDS per operation: with eight, reads and
// arriving loads together keep LDS busy for all of the 2048 clocks that the matrix units take per k-tile.  One wave
// per SIMD has to overlap by itself, so the order of MFMAs, LDS reads and loads is written down, in assembly; the
// accumulators fill the 256 accumulation registers.  A k-tile is two steps of 32 k values, 64 MFMAs each; while one step is
// multiplied the fragments of the next are read, and k-tile t + 2 is loaded into the stage of k-tile t once all waves
// have read all of that.
//   Both operands along k: every MFMA is a piece of assembly, what stands between is the compiler's.
//   k over rows of one or both: the fragments come through transposing reads, in front of which the compiler would wait
//   for all loads.  There a block of 16 MFMAs with the four fragments that it reads, and the wait for them, is one piece.
//
// bfloat16, 4096 x 28672 outputs over 4096: 725 us, 1327 TFLOP/s (eight waves: 820 us), its gradients 723 and 766; 8192 x 4096
// over 14336 with a residual 728 us, its gradients 771 and 773 (medians; the clocks under this load differ by 10 % from call to
// call).  The matrix units work for 68 % of the clocks; k-tiles of MFMAs alone would take 2048 clocks of 2950.  Reads spread
// over 48 MFMAs instead of 32, loads every third MFMA instead of every fifth, blocks of 32 MFMAs, and workgroups that
// load their next tile during the epilogue made no difference or a slower one; 32 x 32 x 16 MFMAs 4 % slower.
#define OPMX_WIDE_ROWS(OP)                                                                                            \
    asm volatile("s_nop 1\n\t"                                                                                        \
                 "v_mfma_f32_16x16x32_" OP " %0, %20, %24, %0\n\t"                                                    \
                 "ds_read_b128 %16, %28 offset:%29\n\t"                                                               \
                 "v_mfma_f32_16x16x32_" OP " %1, %21, %24, %1\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %2, %22, %24, %2\n\t"                                                    \
                 "ds_read_b128 %17, %28 offset:%30\n\t"                                                               \
                 "v_mfma_f32_16x16x32_" OP " %3, %23, %24, %3\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %4, %20, %25, %4\n\t"                                                    \
                 "ds_read_b128 %18, %28 offset:%31\n\t"                                                               \
                 "v_mfma_f32_16x16x32_" OP " %5, %21, %25, %5\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %6, %22, %25, %6\n\t"                                                    \
                 "ds_read_b128 %19, %28 offset:%32\n\t"                                                               \
                 "v_mfma_f32_16x16x32_" OP " %7, %23, %25, %7\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %8, %20, %26, %8\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %9, %21, %26, %9\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %10, %22, %26, %10\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %11, %23, %26, %11\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %12, %20, %27, %12\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %13, %21, %27, %13\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %14, %22, %27, %14\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %15, %23, %27, %15\n\t"                                                  \
                 "s_waitcnt lgkmcnt(0)"                                                                               \
                 : "+a"(acc[PH * 4 + 0][QH * 4 + 0]), "+a"(acc[PH * 4 + 1][QH * 4 + 0]), "+a"(acc[PH * 4 + 2][QH * 4  \
                 + 0]), "+a"(acc[PH * 4 + 3][QH * 4 + 0]), "+a"(acc[PH * 4 + 0][QH * 4 + 1]), "+a"(acc[PH * 4 + 1][QH \
                 * 4 + 1]), "+a"(acc[PH * 4 + 2][QH * 4 + 1]), "+a"(acc[PH * 4 + 3][QH * 4 + 1]), "+a"(acc[PH * 4 +   \
                 0][QH * 4 + 2]), "+a"(acc[PH * 4 + 1][QH * 4 + 2]), "+a"(acc[PH * 4 + 2][QH * 4 + 2]), "+a"(acc[PH * \
                 4 + 3][QH * 4 + 2]), "+a"(acc[PH * 4 + 0][QH * 4 + 3]), "+a"(acc[PH * 4 + 1][QH * 4 + 3]),           \
                 "+a"(acc[PH * 4 + 2][QH * 4 + 3]), "+a"(acc[PH * 4 + 3][QH * 4 + 3]), "=&v"(f[F0 + 0]), "=&v"(f[F0 + \
                 1]), "=&v"(f[F0 + 2]), "=&v"(f[F0 + 3])                                                              \
                 : "v"(p[PH * 4 + 0]), "v"(p[PH * 4 + 1]), "v"(p[PH * 4 + 2]), "v"(p[PH * 4 + 3]), "v"(q[QH * 4 +     \
                 0]), "v"(q[QH * 4 + 1]), "v"(q[QH * 4 + 2]), "v"(q[QH * 4 + 3]), "v"(at[0]), "n"((F0 + 0) * 2048),   \
                 "n"((F0 + 1) * 2048), "n"((F0 + 2) * 2048), "n"((F0 + 3) * 2048)                                     \
                 : "memory")
#define OPMX_WIDE_COLUMNS(OP)                                                                                         \
    asm volatile("s_nop 1\n\t"                                                                                        \
                 "v_mfma_f32_16x16x32_" OP " %0, %24, %28, %0\n\t"                                                    \
                 "ds_read_b64_tr_b16 %16, %32 offset:%36\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %1, %25, %28, %1\n\t"                                                    \
                 "ds_read_b64_tr_b16 %17, %32 offset:%37\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %2, %26, %28, %2\n\t"                                                    \
                 "ds_read_b64_tr_b16 %18, %33 offset:%36\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %3, %27, %28, %3\n\t"                                                    \
                 "ds_read_b64_tr_b16 %19, %33 offset:%37\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %4, %24, %29, %4\n\t"                                                    \
                 "ds_read_b64_tr_b16 %20, %34 offset:%36\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %5, %25, %29, %5\n\t"                                                    \
                 "ds_read_b64_tr_b16 %21, %34 offset:%37\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %6, %26, %29, %6\n\t"                                                    \
                 "ds_read_b64_tr_b16 %22, %35 offset:%36\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %7, %27, %29, %7\n\t"                                                    \
                 "ds_read_b64_tr_b16 %23, %35 offset:%37\n\t"                                                         \
                 "v_mfma_f32_16x16x32_" OP " %8, %24, %30, %8\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %9, %25, %30, %9\n\t"                                                    \
                 "v_mfma_f32_16x16x32_" OP " %10, %26, %30, %10\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %11, %27, %30, %11\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %12, %24, %31, %12\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %13, %25, %31, %13\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %14, %26, %31, %14\n\t"                                                  \
                 "v_mfma_f32_16x16x32_" OP " %15, %27, %31, %15\n\t"                                                  \
                 "s_waitcnt lgkmcnt(0)"                                                                               \
                 : "+a"(acc[PH * 4 + 0][QH * 4 + 0]), "+a"(acc[PH * 4 + 1][QH * 4 + 0]), "+a"(acc[PH * 4 + 2][QH * 4  \
                 + 0]), "+a"(acc[PH * 4 + 3][QH * 4 + 0]), "+a"(acc[PH * 4 + 0][QH * 4 + 1]), "+a"(acc[PH * 4 + 1][QH \
                 * 4 + 1]), "+a"(acc[PH * 4 + 2][QH * 4 + 1]), "+a"(acc[PH * 4 + 3][QH * 4 + 1]), "+a"(acc[PH * 4 +   \
                 0][QH * 4 + 2]), "+a"(acc[PH * 4 + 1][QH * 4 + 2]), "+a"(acc[PH * 4 + 2][QH * 4 + 2]), "+a"(acc[PH * \
                 4 + 3][QH * 4 + 2]), "+a"(acc[PH * 4 + 0][QH * 4 + 3]), "+a"(acc[PH * 4 + 1][QH * 4 + 3]),           \
                 "+a"(acc[PH * 4 + 2][QH * 4 + 3]), "+a"(acc[PH * 4 + 3][QH * 4 + 3]), "=&v"(v[0]), "=&v"(v[1]),      \
                 "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])                         \
                 : "v"(p[PH * 4 + 0]), "v"(p[PH * 4 + 1]), "v"(p[PH * 4 + 2]), "v"(p[PH * 4 + 3]), "v"(q[QH * 4 +     \
                 0]), "v"(q[QH * 4 + 1]), "v"(q[QH * 4 + 2]), "v"(q[QH * 4 + 3]), "v"(at[0]), "v"(at[1]), "v"(at[2]), \
                 "v"(at[3]), "n"(KS * 16384), "n"(KS * 16384 + 2048)                                                  \
                 : "memory")

// acc[PH * 4 + j][QH * 4 + i] += p[PH * 4 + j] q[QH * 4 + i], and the fragments F0 ... F0 + 3 of the next step into f.  KM:
// from a k-major tile, at[0 ... 3] their LDS addresses at k step 0; else at[0] the address of fragment 0 at the step.
// The two wait states in front: the compiler may have moved a fragment just before, and does not see MFMAs in assembly.
#define OPMX_WIDE_BLOCK(T, OP)                                                                                        \
    template <int PH, int QH, int F0, bool KM, int KS>                                                                \
    __device__ __forceinline__ void wide_block(float4_t (&acc)[8][8], const Step<T>::frag (&p)[8],                    \
                                               const Step<T>::frag (&q)[8], Step<T>::frag (&f)[8], const uint32_t *at) \
    {                                                                                                                 \
        if constexpr (KM) {                                                                                           \
            u32pair v[8];                                                                                             \
            OPMX_WIDE_COLUMNS(OP);                                                                                    \
            _Pragma("unroll") for (int j = 0; j < 4; ++j) __builtin_memcpy(&f[F0 + j], &v[2 * j], 16);                \
        } else {                                                                                                      \
            OPMX_WIDE_ROWS(OP);                                                                                       \
        }                                                                                                             \
    }
OPMX_WIDE_BLOCK(f16, "f16")
OPMX_WIDE_BLOCK(bf16, "bf16")

// LDS addresses of a lane's fragments of one operand: first = the wave's first row / 16 (a multiple of 8), base = the
// tile's address.
template <bool KM> struct WideReader {
    uint32_t a[KM ? 8 : 2];
    __device__ __forceinline__ void init(uint32_t base, int first, int lane)
    {
        const int r = lane & 15, g = lane >> 4;
        if constexpr (KM) {
            const int k = g * 8 + (r >> 2);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                a[i] = base + k * 512 + (((first + i) ^ unit_swizzle<f16, 256>(k)) << 5) + (r & 3) * 8;
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) a[ks] = base + (first * 16 + r) * kTileBytes + (((ks * 4 + g) ^ ((r >> 1) & 7)) << 4);
        }
    }
    // for the fragments F0 ... F0 + 3 of k step KS in the stage at `stage` bytes
    template <int F0, int KS> __device__ __forceinline__ void at(uint32_t stage, uint32_t (&out)[4]) const
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = (KM ? a[KM ? F0 + i : 0] : a[KM ? 0 : KS]) + stage;
    }
};

template <typename T, bool PK, bool QK, bool GATED>
__global__ __launch_bounds__(256, 1) void linear_gemm_wide_kernel(Operand P, Operand Q, int64_t Kc, Epilogue e, uint32_t mt,
                                                                  uint32_t nt)
{
    constexpr int BM = 256, BN = 256, STAGE = (BM + BN) * kTileBytes, BK = kTileBytes / sizeof(T);
    using frag = typename Step<T>::frag;
    extern __shared__ __attribute__((aligned(16))) char smem[];

    int64_t tm, tc;
    place(blockIdx.x, mt, nt, tm, tc);
    const int64_t m0 = tm * BM, c0 = tc * (GATED ? BN / 2 : BN);
    const int nk = static_cast<int>((Kc + BK - 1) / BK);
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wm = wave >> 1, wn = wave & 1;

    Loader<T, BN, 256, PK, GATED> lp;
    Loader<T, BM, 256, QK, false> lq;
    lp.init(P, c0, e.ncols, 0);
    lq.init(Q, m0, e.rows, 0);
    WideReader<PK> rp;
    WideReader<QK> rq;
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(OPMX_LDS(smem)));
    rp.init(lds + BM * kTileBytes, wn * 8, lane);
    rq.init(lds, wm * 8, lane);

    float4_t acc[8][8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[j][i] = float4_t{0.f, 0.f, 0.f, 0.f};

    int64_t k_left = Kc;
    // pieces [4 Q4, 4 Q4 + 4) of the sixteen of the next k-tile to be loaded
    auto load4 = [&](char *stage, auto q4) {
        constexpr int Q4 = decltype(q4)::value;
        const int left = k_left < BK ? static_cast<int>(k_left) : BK;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (Q4 < 2) lq.issue(Q4 * 4 + i, stage, left);
            else lp.issue((Q4 - 2) * 4 + i, stage + BM * kTileBytes, left);
        }
        if constexpr (Q4 == 3) {
            lq.next();
            lp.next();
            k_left -= BK;
        }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        char *stage = smem + t * STAGE;
        load4(stage, I0{});
        load4(stage, I1{});
        load4(stage, I2{});
        load4(stage, I3{});
    }
    wait_loads<16>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    frag pa[8], qa[8], pb[8], qb[8];                     // of step 0 and of step 1
    fragments<T, BN, PK, 0, 8>(smem + BM * kTileBytes, wn * 8, lane, pa);
    fragments<T, BM, QK, 0, 8>(smem, wm * 8, lane, qa);

    // The wait states between the last MFMA and the first use of an accumulator, at the end of every k-tile: the compiler does
    // not know of the MFMAs, and copies accumulators as soon as the loop is left, in front of any wait that stands there.
    auto retire = [] { asm volatile("s_nop 11" ::: "memory"); };
    uint32_t cur = 0, at[4];
    if constexpr (!PK && !QK) {
        // Step 0 reads the other step's fragments behind its first 32 MFMAs.  After the 40th all waves have them: the stage
        // is free, and the 16 loads of k-tile t + 2 go out behind every fifth MFMA from there on.  In the middle of step 1
        // (11 of them are out) the loads of k-tile t + 1 must have landed, one and a half k-tiles after they went out.
        const char *p0 = smem + BM * kTileBytes, *q0 = smem;
        const int r = lane & 15, g = lane >> 4;
        const int slot[2] = {(g ^ ((r >> 1) & 7)) << 4, ((4 + g) ^ ((r >> 1) & 7)) << 4};
        const int rowp = (wn * 128 + r) * kTileBytes, rowq = (wm * 128 + r) * kTileBytes;
        auto read = [&](uint32_t stage, int ks, int i, frag (&p)[8], frag (&q)[8]) {
            if (i < 8) p[i < 8 ? i : 0] = *reinterpret_cast<const frag *>(p0 + stage + rowp + slot[ks] + (i & 7) * 16 * kTileBytes);
            else q[i < 8 ? 0 : i - 8] = *reinterpret_cast<const frag *>(q0 + stage + rowq + slot[ks] + (i & 7) * 16 * kTileBytes);
        };
        for (int kt = 0; kt < nk; ++kt) {
            const int left = k_left < BK ? static_cast<int>(k_left) : BK;
            char *free_stage = smem + cur;
            auto load1 = [&](int i) {
                if (i < 8) lq.issue(i < 8 ? i : 0, free_stage, left);
                else lp.issue(i < 8 ? 0 : i - 8, free_stage + BM * kTileBytes, left);
            };
#pragma unroll
            for (int m = 0; m < 64; ++m) {
                Mfma<T>::m16_acc(pa[m % 8], qa[m / 8], acc[m % 8][m / 8]);
                if (m < 32 && m % 2 == 0) read(cur, 1, m / 2, pb, qb);
                if (m == 40) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                if (m > 40 && (m - 41) % 5 == 0) load1((m - 41) / 5);
            }
#pragma unroll
            for (int m = 0; m < 64; ++m) {
                Mfma<T>::m16_acc(pb[m % 8], qb[m / 8], acc[m % 8][m / 8]);
                if (m == 32) {
                    asm volatile("s_waitcnt vmcnt(11)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                if (m < 53 && (m - 2) % 5 == 0) load1(5 + (m - 2) / 5);
                if (m > 32 && m % 2 == 1) read(cur ^ STAGE, 0, (m - 33) / 2, pa, qa);
            }
            retire();
            lq.next();
            lp.next();
            k_left -= BK;
            cur ^= STAGE;
        }
    } else {
        // Step 0 (pa, qa) reads the fragments of step 1 from the same stage; then the wave waits for its loads of k-tile t + 1
        // (issued a k-tile ago) and for the other waves, and step 1 reads the first fragments of k-tile t + 1 from the other
        // stage while k-tile t + 2 is loaded into this one.
        for (int kt = 0; kt < nk; ++kt) {
            rp.template at<0, 1>(cur, at);
            wide_block<0, 0, 0, PK, 1>(acc, pa, qa, pb, at);
            rp.template at<4, 1>(cur, at);
            wide_block<1, 0, 4, PK, 1>(acc, pa, qa, pb, at);
            rq.template at<0, 1>(cur, at);
            wide_block<0, 1, 0, QK, 1>(acc, pa, qa, qb, at);
            rq.template at<4, 1>(cur, at);
            wide_block<1, 1, 4, QK, 1>(acc, pa, qa, qb, at);

            wait_loads<0>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");

            char *free_stage = smem + cur;
            cur ^= STAGE;
            load4(free_stage, I0{});
            rp.template at<0, 0>(cur, at);
            wide_block<0, 0, 0, PK, 0>(acc, pb, qb, pa, at);
            load4(free_stage, I1{});
            rp.template at<4, 0>(cur, at);
            wide_block<1, 0, 4, PK, 0>(acc, pb, qb, pa, at);
            load4(free_stage, I2{});
            rq.template at<0, 0>(cur, at);
            wide_block<0, 1, 0, QK, 0>(acc, pb, qb, qa, at);
            load4(free_stage, I3{});
            rq.template at<4, 0>(cur, at);
            wide_block<1, 1, 4, QK, 0>(acc, pb, qb, qa, at);
            retire();
        }
    }
    wait_loads<0>();                                     // the epilogue uses the same memory
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    write_columns<T, 8, 8, GATED>(acc, e, m0 + wm * 128, c0 + wn * (GATED ? 64 : 128), lane, smem + wave * (64 * 256));
}

template <typename T, bool PK, bool QK, bool GATED>
int launch_wide(const Operand &P, const Operand &Q, int64_t Kc, const Epilogue &e, hipStream_t s)
{
    constexpr int SMEM = 2 * 512 * kTileBytes;
    const int64_t mt = ceil_div(e.rows, 256), nt = ceil_div(e.ncols, GATED ? 128 : 256);
    if (mt * nt == 0) return OPMX_OK;
    if (mt * nt >= (int64_t{1} << 31)) return OPMX_ERR_UNSUPPORTED;
    static std::atomic<uint64_t> done{0};
    const void *k = reinterpret_cast<const void *>(&linear_gemm_wide_kernel<T, PK, QK, GATED>);
    if (!ensure_dynamic_smem(k, SMEM, done)) return OPMX_ERR_LAUNCH;
    linear_gemm_wide_kernel<T, PK, QK, GATED><<<static_cast<unsigned>(mt * nt), 256, SMEM, s>>>(
        P, Q, Kc, e, static_cast<uint32_t>(mt), static_cast<uint32_t>(nt));
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

template <typename T> int by_layout_wide(const Operand &P, const Operand &Q, int64_t Kc, const Epilogue &e, hipStream_t s)
{
    if (e.act == OPMX_ACTIVATION_SWIGLU) return launch_wide<T, false, false, true>(P, Q, Kc, e, s);
    if (!P.k_major) return launch_wide<T, false, false, false>(P, Q, Kc, e, s);
    if (!Q.k_major) return launch_wide<T, true, false, false>(P, Q, Kc, e, s);
    return launch_wide<T, true, true, false>(P, Q, Kc, e, s);
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES, bool PK, bool QK, bool GATED>
int launch(const Operand &P, const Operand &Q, int64_t Kc, const Epilogue &e, int ranges, hipStream_t s)
{
    constexpr int BNO = GATED ? BN / 2 : BN, BK = kTileBytes / sizeof(T), SMEM = STAGES * (BM + BN) * kTileBytes;
    const int64_t mt = ceil_div(e.rows, BM), nt = ceil_div(e.ncols, BNO), nk = ceil_div(Kc, BK);
    const int64_t per = nk > 0 ? ceil_div(nk, ranges) : 1;
    const int64_t used = nk > 0 ? ceil_div(nk, per) : 1;    // every range holds at least one k-tile
    if (mt * nt == 0) return OPMX_OK;
    if (mt * nt >= (int64_t{1} << 31) || used > 65535 || (ranges > 1 && used != ranges)) return OPMX_ERR_UNSUPPORTED;
    static std::atomic<uint64_t> done{0};
    const void *k = reinterpret_cast<const void *>(&linear_gemm_kernel<T, BM, BN, WM, WN, STAGES, PK, QK, GATED>);
    if (!ensure_dynamic_smem(k, SMEM, done)) return OPMX_ERR_LAUNCH;
    linear_gemm_kernel<T, BM, BN, WM, WN, STAGES, PK, QK, GATED>
        <<<dim3(static_cast<unsigned>(mt * nt), static_cast<unsigned>(used)), WM * WN * kWave, SMEM, s>>>(
            P, Q, Kc, e, static_cast<uint32_t>(mt), static_cast<uint32_t>(nt), per);
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

template <typename T, int BM, int BN, int WM, int WN, int STAGES>
int by_layout(const Operand &P, const Operand &Q, int64_t Kc, const Epilogue &e, int ranges, hipStream_t s)
{
    if (e.act == OPMX_ACTIVATION_SWIGLU) return launch<T, BM, BN, WM, WN, STAGES, false, false, true>(P, Q, Kc, e, ranges, s);
    if (!P.k_major) return launch<T, BM, BN, WM, WN, STAGES, false, false, false>(P, Q, Kc, e, ranges, s);
    if (!Q.k_major) return launch<T, BM, BN, WM, WN, STAGES, true, false, false>(P, Q, Kc, e, ranges, s);
    return launch<T, BM, BN, WM, WN, STAGES, true, true, false>(P, Q, Kc, e, ranges, s);
}

template <typename T> int by_tile(const Operand &P, const Operand &Q, int64_t Kc, const Epilogue &e, Tile tile, int ranges, hipStream_t s)
{
    switch (tile) {
        case Tile::k256:
            if constexpr (sizeof(T) == 2)
                if (ranges == 1) return by_layout_wide<T>(P, Q, Kc, e, s);
            break;
        case Tile::k128: return by_layout<T, 128, 128, 2, 2, 2>(P, Q, Kc, e, ranges, s);
        case Tile::k64: return by_layout<T, 64, 128, 2, 2, 3>(P, Q, Kc, e, ranges, s);
        case Tile::k32:
            if constexpr (sizeof(T) == 4) return by_layout<T, 32, 128, 2, 2, 3>(P, Q, Kc, e, ranges, s);
            break;
    }
    return OPMX_ERR_UNSUPPORTED;
}

}  // namespace

int launch_linear_gemm(const Operand &P, const Operand &Q, int64_t Kc, int dtype, const Epilogue &e, Tile tile, int ranges,
                       hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return by_tile<float>(P, Q, Kc, e, tile, ranges, s);
        case OPMX_DTYPE_F16: return by_tile<f16>(P, Q, Kc, e, tile, ranges, s);
        case OPMX_DTYPE_BF16: return by_tile<bf16>(P, Q, Kc, e, tile, ranges, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

}  // namespace opmx
