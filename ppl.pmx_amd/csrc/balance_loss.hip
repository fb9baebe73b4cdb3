// Balance loss of the router and tokens per expert, with the gradient.
//
//   p[t, :] = softmax(scores[t, :]);  count[e] = kept tokens with e among their k largest scores;
//   f = count / (k n), n kept tokens;  loss = E sum_e f_e (1/n) sum_t p[t, e];
//   w_e = E f_e / n (held constant):  dscores[t, e] = dloss p[t, e] (w_e - sum_j w_j p[t, j]).
//
// The picks are MoeSelect's (ties to the lower expert id, NaN ranks first, -0 equals +0), so count is the
// difference of its expert_offset.  A row of -inf alone has p = 0: it has nothing to spread.
//
// Scores are read once in each direction and the gradient is written once.  A token belongs to L lanes (a power of two, a
// constant of the kernel), each of which holds V of its E scores in registers.  A lane meets the same V experts in every token, so sums over tokens stay in registers until the block is done.  The k-th largest score
// comes from lists, not from k rounds of a wave-wide maximum: every lane keeps the KL largest of its keys sorted
// (one median-of-three per slot and key) and the lists of the L lanes meet in log2 L bitonic
// merges.  131072 tokens, 256 experts, k = 8, fp32: forward 50 us (bound by instructions; the scores alone would take 22) and
// 7 for the blocks' sums, backward 44 us, 6.1 TB/s.
// An expert is picked where its key is not below the k-th; keys of 16-bit scores hold the id too and are
// distinct, equal fp32 scores at the k-th place are settled by id in a branch few waves take.
// Sums of p: fp32 over up to kFold tokens of a lane and over the lanes of the block, 64 bits beyond, in a fixed order: results
// do not vary, and what a sum is off by does not grow with the number of tokens.
#include "train.h"

namespace opmx {
namespace {

constexpr int kMaxBlocks = 256;
constexpr int kFold = 64;       // tokens of a lane whose p are added in fp32
__host__ __device__ inline int pitch_of(int E) { return (E + 3) / 4 * 4; }      // of a block's sums

// A key orders scores as MoeSelect does: NaN first, -0 equal to +0.  No key is 0 or 2^32 - 1.
template <typename T> struct Key {
    static constexpr bool unique = true;     // 16 bits of score, 16 bits of id
    static __device__ __forceinline__ uint32_t of(T v, int id)
    {
        uint16_t b;
        __builtin_memcpy(&b, &v, 2);
        uint32_t u = b;
        u = u == 0x8000u ? 0u : u;
        u ^= (u & 0x8000u) ? 0xFFFFu : 0x8000u;
        u = v != v ? 0xFFFEu : u;
        return (u << 16) | (0xFFFFu - static_cast<uint32_t>(id));
    }
};
template <> struct Key<float> {
    static constexpr bool unique = false;
    static __device__ __forceinline__ uint32_t of(float f, int)
    {
        const uint32_t u = __float_as_uint(f + 0.0f);
        const uint32_t key = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
        return f != f ? 0xFFFFFFFEu : key;
    }
};

// Exchanges inside rows of 16 lanes are register moves (DPP); only those across rows go through LDS.
template <int CTRL, typename U> __device__ __forceinline__ U dpp(U v)
{
    int b;
    __builtin_memcpy(&b, &v, 4);
    b = __builtin_amdgcn_update_dpp(0, b, CTRL, 0xF, 0xF, true);
    U r;
    __builtin_memcpy(&r, &b, 4);
    return r;
}
// The value of a lane of the other half of a group of 2 D lanes, when all lanes of a half hold the same.
template <int D, typename U> __device__ __forceinline__ U other_half(U v)
{
    if constexpr (D == 1) return dpp<0xB1>(v);          // quad_perm 1,0,3,2
    else if constexpr (D == 2) return dpp<0x4E>(v);     // quad_perm 2,3,0,1
    else if constexpr (D == 4) return dpp<0x141>(v);    // row_half_mirror
    else if constexpr (D == 8) return dpp<0x140>(v);    // row_mirror
    else return __shfl_xor(v, D, kWave);
}
// The value D lanes before in a group, 0 for the group's first D lanes.
template <int D, int L> __device__ __forceinline__ int lanes_before(int v, int lane)
{
    int o;
    if constexpr (L <= 16) o = dpp<0x110 + D>(v);       // row_shr D: a group lies within a row of 16 lanes
    else o = __shfl_up(v, D, kWave);
    return lane >= D ? o : 0;
}
// Sum over the lanes that are equal mod L (a power of two), in every one of them.
template <int L, typename U> __device__ __forceinline__ U sum_mod(U v)
{
    if (L <= 1) v += dpp<0xB1>(v);
    if (L <= 2) v += dpp<0x4E>(v);
    if (L <= 4) v += dpp<0x124>(v);                     // row_ror 4: lanes i and i + 4, then
    if (L <= 8) v += dpp<0x128>(v);                     // row_ror 8: the other two of the four
    if (L <= 16) v += __shfl_xor(v, 16, kWave);
    if (L <= 32) v += __shfl_xor(v, 32, kWave);
    return v;
}
// f(D) for D = 1, 2, ... below L (a constant).
#define OPMX_HALVES(f)               \
    do {                             \
        if constexpr (L > 1) f(1);   \
        if constexpr (L > 2) f(2);   \
        if constexpr (L > 4) f(4);   \
        if constexpr (L > 8) f(8);   \
        if constexpr (L > 16) f(16); \
    } while (0)

__device__ __forceinline__ uint32_t umax_(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin_(uint32_t a, uint32_t b) { return a < b ? a : b; }

// The id of a lane's i-th score: chunks of N consecutive ids go round the L lanes of the token.
template <int N, int L> __device__ __forceinline__ int expert_of(int i, int lane) { return ((i / N) * L + lane) * N + i % N; }

// A lane's V scores of a token as floats; experts past E, and all of a token that does not count, read as -inf.  keys
// (KEYS) get 0 there.
template <typename T, int N, int V, int L, bool KEYS>
__device__ __forceinline__ void load_scores(const T *__restrict__ row, int E, int lane, bool keep, float (&z)[V],
                                            uint32_t (&key)[KEYS ? V : 1])
{
    T v[V];
#pragma unroll
    for (int c = 0; c < V / N; ++c) {        // E % N == 0: a chunk is whole or absent, and then the last one is read
        const int e0 = (c * L + lane) * N, at = e0 < E ? e0 : E - N;
        if constexpr (N == 1) v[c] = row[at];
        else {
            const Vec16<T> q = load16_once(row + at);
#pragma unroll
            for (int j = 0; j < N; ++j) v[c * N + j] = q.v[j];
        }
    }
#pragma unroll
    for (int c = 0; c < V / N; ++c) {
        const int e0 = (c * L + lane) * N;
        const bool in = keep && e0 < E;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = c * N + j;
            z[i] = in ? to_f32(v[i]) : -INFINITY;
            if constexpr (KEYS) key[i] = in ? Key<T>::of(v[i], e0 + j) : 0u;
        }
    }
}

// z -> e^(z - max) over the token's L lanes; the value returned takes them to the softmax.  The hardware's exp2: z - max and its
// product with log2 e are off by |z - max| 2^-24 each, so is the result, plus an ulp.  (One fma of z would do, but not
// for masks of the type's lowest value.)  A row of -inf alone gives 0; a NaN or an infinity makes all of the row NaN.
template <int V, int L> __device__ __forceinline__ float exp_(float (&z)[V])
{
    constexpr float kLog2e = 1.44269504088896341f;
    float m = z[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, z[i]);
#define OPMX_MAX(D) m = fmaxf(m, other_half<D>(m))
    OPMX_HALVES(OPMX_MAX);
    const bool nothing = m == -INFINITY;
    m = nothing ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        z[i] = __builtin_amdgcn_exp2f((z[i] - m) * kLog2e);
        sum += z[i];
    }
#define OPMX_SUM(D) sum += other_half<D>(sum)
    OPMX_HALVES(OPMX_SUM);
    return nothing ? 0.0f : __builtin_amdgcn_rcpf(sum);
}

// Inserts x into the list a[0] >= a[1] >= ..., dropping the smallest.
template <int KL> __device__ __forceinline__ void insert(uint32_t (&a)[KL], uint32_t x)
{
#pragma unroll
    for (int j = KL - 1; j >= 1; --j)            // the median of x, a[j-1] >= a[j], in the form of v_med3_u32
        a[j] = umax_(umin_(x, a[j - 1]), umin_(umax_(x, a[j - 1]), a[j]));
    a[0] = umax_(a[0], x);
}

// a: the KL largest of a's and the other half's lists, sorted again.
template <int KL, int D> __device__ __forceinline__ void merge(uint32_t (&a)[KL])
{
    uint32_t b[KL];
#pragma unroll
    for (int j = 0; j < KL; ++j) b[j] = other_half<D>(a[KL - 1 - j]);
#pragma unroll
    for (int j = 0; j < KL; ++j) a[j] = umax_(a[j], b[j]);                      // bitonic
#pragma unroll
    for (int h = KL / 2; h >= 1; h >>= 1)
#pragma unroll
        for (int j = 0; j < KL; ++j)
            if ((j & h) == 0) {
                const uint32_t hi = umax_(a[j], a[j + h]), lo = umin_(a[j], a[j + h]);
                a[j] = hi;
                a[j + h] = lo;
            }
}

// a[i] of a descending list, as a maximum over a[i], a[i+1], ...: a selection by index would put the list into LDS,
// at an address that every workgroup works out from the dispatch packet in host memory (57 ns each, one after the other:
// 15 us of a launch of 256).
template <int KL> __device__ __forceinline__ uint32_t at(const uint32_t (&a)[KL], int i)
{
    uint32_t v = 0u;
#pragma unroll
    for (int j = 0; j < KL; ++j) v = umax_(v, j >= i ? a[j] : 0u);
    return v;
}

// What the sums over tokens become: loss, counts, and w for the backward pass.  One block.
template <int THREADS>
__device__ __forceinline__ void finish(double psum, int64_t count, int64_t kept, int e, int E, int k, double *red,
                                       float *loss, int64_t *counts, float *w)
{
    const double n = kept > 0 ? static_cast<double>(kept) : 1.0;
    double part = 0.0;
    if (e < E) {
        const double weight = static_cast<double>(E) * static_cast<double>(count) / (static_cast<double>(k) * n * n);   // E f / n
        part = weight * psum;
        counts[e] = count;
        w[e] = static_cast<float>(weight);
    }
    // E <= 256 values lie in the first four waves
    for (int d = 1; d < kWave; d <<= 1) part += __shfl_xor(part, d, kWave);
    if (lane_id() == 0 && threadIdx.x < OPMX_MOE_MAX_EXPERTS) red[threadIdx.x / kWave] = part;
    __syncthreads();
    if (threadIdx.x == 0) {
        double v = red[0];
        for (int i = 1; i < THREADS / kWave && i < OPMX_MOE_MAX_EXPERTS / kWave; ++i) v += red[i];
        *loss = static_cast<float>(v);
    }
}

// Sums over the tokens of a block.  A single block finishes by itself; several leave psum and counts
// [blocks][pitch_of(E)] and kept [blocks] in the workspace.
template <typename T, int N, int V, int L, int KL, int THREADS>
__global__ __launch_bounds__(THREADS) void balance_kernel(const T *__restrict__ scores,
                                                           const uint8_t *__restrict__ mask, int64_t Ttok, int E, int k,
                                                           float *__restrict__ part_p, int32_t *__restrict__ part_c,
                                                           int32_t *__restrict__ part_n, float *__restrict__ loss,
                                                           int64_t *__restrict__ counts, float *__restrict__ w)
{
    constexpr int WAVES = THREADS / kWave;
    __shared__ float s_p[WAVES][OPMX_MOE_MAX_EXPERTS];
    __shared__ int32_t s_c[WAVES][OPMX_MOE_MAX_EXPERTS];
    __shared__ int32_t s_n[WAVES];
    __shared__ double s_red[OPMX_MOE_MAX_EXPERTS / kWave];
    const int lane = lane_id() % L, wave = threadIdx.x / kWave;
    const int per_block = THREADS / L;
    float psum[V];
    int32_t cnt[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        psum[i] = 0.0f;
        cnt[i] = 0;
    }
    int32_t kept = 0;
    int64_t t0 = static_cast<int64_t>(blockIdx.x) * per_block;
    const int e = threadIdx.x;
    double p = 0.0;                              // of expert e, of the block
    int32_t c = 0, n = 0;
    while (true) {
        for (int trip = 0; trip < kFold && t0 < Ttok; ++trip, t0 += static_cast<int64_t>(gridDim.x) * per_block) {
            const int64_t t = t0 + threadIdx.x / L;
            const bool keep = t < Ttok && (mask == nullptr || mask[t] != 0);     // the same in the token's L lanes
            const T *row = scores + (t < Ttok ? t : Ttok - 1) * E;
            float z[V];
            uint32_t key[V];
            load_scores<T, N, V, L, true>(row, E, lane, keep, z, key);
            uint32_t list[KL];
#pragma unroll
            for (int j = 0; j < KL; ++j) list[j] = 0u;
#pragma unroll
            for (int i = 0; i < V; ++i) insert<KL>(list, key[i]);
#define OPMX_MERGE(D) merge<KL, D>(list)
            OPMX_HALVES(OPMX_MERGE);
            const uint32_t kth = keep ? at<KL>(list, k - 1) : 0xFFFFFFFFu;       // no key of a token that does not count reaches it
            bool tied = false;
            if constexpr (!Key<T>::unique) {
                int picked = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) picked += key[i] >= kth ? 1 : 0;
#define OPMX_PICKED(D) picked += other_half<D>(picked)
                OPMX_HALVES(OPMX_PICKED);
                tied = picked > k;               // more equal ones at the k-th place than are to be picked
            }
            if (!__any(tied)) {
#pragma unroll
                for (int i = 0; i < V; ++i) cnt[i] += key[i] >= kth ? 1 : 0;
            } else {
                int above = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) above += key[i] > kth ? 1 : 0;
#define OPMX_ABOVE(D) above += other_half<D>(above)
                OPMX_HALVES(OPMX_ABOVE);
                const int left = k - above;      // so many of the equal ones are picked, the lowest ids first
                // ids go up chunk by chunk, and within a chunk lane by lane
                int before = 0;                  // equal ones in the chunks behind us
#pragma unroll
                for (int c = 0; c < V / N; ++c) {
                    int mine = 0;
#pragma unroll
                    for (int j = 0; j < N; ++j) mine += key[c * N + j] == kth ? 1 : 0;
                    int upto = mine, all = mine;
#define OPMX_PREFIX(D) upto += lanes_before<D, L>(upto, lane), all += other_half<D>(all)
                    OPMX_HALVES(OPMX_PREFIX);
                    int rank = before + upto - mine;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const uint32_t q = key[c * N + j];
                        cnt[c * N + j] += q > kth || (q == kth && rank < left) ? 1 : 0;
                        rank += q == kth ? 1 : 0;
                    }
                    before += all;
                }
            }
            const float scale = exp_<V, L>(z);
#pragma unroll
            for (int i = 0; i < V; ++i) psum[i] = fmaf(z[i], scale, psum[i]);
            kept += keep && lane == 0 ? 1 : 0;
        }
        // over the tokens of the wave, then of the block
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float ps = sum_mod<L>(psum[i]);
            const int32_t cs = sum_mod<L>(cnt[i]);
            psum[i] = 0.0f;
            cnt[i] = 0;
            const int id = expert_of<N, L>(i, lane);
            if (lane_id() < L && id < E) {
                s_p[wave][id] = ps;
                s_c[wave][id] = cs;
            }
        }
        kept = sum_mod<1>(kept);
        if (lane_id() == 0) s_n[wave] = kept;
        kept = 0;
        __syncthreads();
        if (e < E) {
            float part = 0.0f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
                part += s_p[v][e];
                c += s_c[v][e];
            }
            p += part;
        }
#pragma unroll
        for (int v = 0; v < WAVES; ++v) n += s_n[v];
        if (t0 >= Ttok) break;
        __syncthreads();                         // before they are written again
    }
    if (gridDim.x == 1) {
        finish<THREADS>(p, c, n, e, E, k, s_red, loss, counts, w);
        return;
    }
    if (e < pitch_of(E)) {                   // (p and c are 0 past E)
        part_p[blockIdx.x * pitch_of(E) + e] = static_cast<float>(p);
        part_c[blockIdx.x * pitch_of(E) + e] = c;
    }
    if (e == 0) part_n[blockIdx.x] = n;
}

// The blocks' sums: a thread adds four experts' of every 16th block, eight blocks' loads in flight, then the slices are
// added in order.  Rows of the sums are pitch_of(E) long: whole 16-byte chunks.
constexpr int kFinish = 1024, kSlices = 16;
__global__ __launch_bounds__(kFinish) void balance_finish_kernel(const float4 *__restrict__ part_p,
                                                                 const int4 *__restrict__ part_c,
                                                                 const int32_t *__restrict__ part_n, int blocks, int E,
                                                                 int k, float *__restrict__ loss,
                                                                 int64_t *__restrict__ counts, float *__restrict__ w)
{
    __shared__ double s_p[kSlices][OPMX_MOE_MAX_EXPERTS];
    __shared__ int32_t s_c[kSlices][OPMX_MOE_MAX_EXPERTS];       // T < 2^31
    __shared__ double s_red[OPMX_MOE_MAX_EXPERTS / kWave];
    __shared__ int32_t s_n;
    const int quads = pitch_of(E) / 4, slice = threadIdx.x / quads, quad = threadIdx.x % quads;
    if (slice < kSlices) {
        double p[4] = {0.0, 0.0, 0.0, 0.0};
        int32_t c[4] = {0, 0, 0, 0};
        for (int b0 = slice; b0 < blocks; b0 += 8 * kSlices) {
            float4 pv[8];
            int4 cv[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {                        // (past the last block the last one again, for nothing)
                const int b = b0 + u * kSlices, at = (b < blocks ? b : blocks - 1) * quads + quad;
                pv[u] = part_p[at];
                cv[u] = part_c[at];
            }
            __builtin_amdgcn_sched_barrier(0);                   // all of them before the first sum
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (b0 + u * kSlices < blocks) {
                    p[0] += pv[u].x, p[1] += pv[u].y, p[2] += pv[u].z, p[3] += pv[u].w;
                    c[0] += cv[u].x, c[1] += cv[u].y, c[2] += cv[u].z, c[3] += cv[u].w;
                }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s_p[slice][quad * 4 + j] = p[j];
            s_c[slice][quad * 4 + j] = c[j];
        }
    }
    if (threadIdx.x >= kFinish - kWave) {
        int32_t n = 0;
#pragma unroll
        for (int b = 0; b < kMaxBlocks; b += kWave) n += b + lane_id() < blocks ? part_n[b + lane_id()] : 0;
        n = sum_mod<1>(n);
        if (lane_id() == 0) s_n = n;
    }
    __syncthreads();
    double p = 0.0;
    int64_t c = 0;
    const int e = threadIdx.x;
    if (e < E)
#pragma unroll
        for (int v = 0; v < kSlices; ++v) {
            p += s_p[v][e];
            c += s_c[v][e];
        }
    finish<kFinish>(p, c, s_n, e, E, k, s_red, loss, counts, w);
}

template <typename T, int N, int V, int L>
__global__ __launch_bounds__(256) void balance_backward_kernel(const T *__restrict__ scores,
                                                               const uint8_t *__restrict__ mask,
                                                               const float *__restrict__ w,
                                                               const float *__restrict__ dloss, int64_t Ttok, int E,
                                                               T *__restrict__ dscores)
{
    const int lane = lane_id() % L, per_block = 256 / L;
    float wv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = expert_of<N, L>(i, lane);
        wv[i] = e < E ? w[e] : 0.0f;
    }
    const float scale = *dloss;
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * per_block; t0 < Ttok;
         t0 += static_cast<int64_t>(gridDim.x) * per_block) {
        const int64_t t = t0 + threadIdx.x / L;
        const bool keep = t < Ttok && (mask == nullptr || mask[t] != 0);
        float z[V];
        uint32_t none[1];
        load_scores<T, N, V, L, false>(scores + (t < Ttok ? t : Ttok - 1) * E, E, lane, keep, z, none);
        const float inverse = exp_<V, L>(z);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            z[i] *= inverse;
            dot += z[i] * wv[i];
        }
#define OPMX_DOT(D) dot += other_half<D>(dot)
        OPMX_HALVES(OPMX_DOT);
        // dot is off by its own rounding and by that of a sum of p that is not quite 1; what is left of the mean of w - dot takes
        // both away.  Where the w are nearly equal (all experts picked by every token) that is all there is.
        float rest = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) rest += z[i] * (wv[i] - dot);
#define OPMX_REST(D) rest += other_half<D>(rest)
        OPMX_HALVES(OPMX_REST);
        if (t >= Ttok) continue;             // (the last trip: nobody needs this lane again)
        T *out = dscores + t * E;
#pragma unroll
        for (int c = 0; c < V / N; ++c) {
            const int e0 = (c * L + lane) * N;
            if (e0 >= E) continue;
            T o[N];
#pragma unroll
            for (int j = 0; j < N; ++j)
                o[j] = from_f32<T>(keep ? scale * z[c * N + j] * ((wv[c * N + j] - dot) - rest) : 0.0f);
            if constexpr (N == 1) out[e0] = o[0];
            else {
                Vec16<T> q;
#pragma unroll
                for (int j = 0; j < N; ++j) q.v[j] = o[j];
                store16(out + e0, q);
            }
        }
    }
}

// Lanes L per token and scores V per lane.  Up to 64 experts a lane holds 8 scores: more lanes per token, and the few
// tokens of a batch spread over more of them; blocks of 4 waves.  Beyond, 16, and blocks of 16 waves: the sums of
// one block per CU are all that the second launch has to add.  L is a constant of the kernels, whose code
// then has no branches.
constexpr int kFewExperts = 64, kFewThreads = 256, kManyThreads = 1024;
constexpr int kFewPicks = 8, kPickThreads = 512;     // more picks: lists of 32 keys leave registers for 8 scores and 8 waves
constexpr int kPickLanesFew = 8, kPickLanesMany = 32;
inline int lanes_few(int E) { return E <= 8 ? 1 : E <= 16 ? 2 : E <= 32 ? 4 : 8; }
inline int lanes_many(int E) { return E <= 128 ? 8 : 16; }

struct Forward {
    const void *scores, *mask;
    int64_t Ttok;
    int E, k, blocks;
    float *pp;
    int32_t *pc, *pn;
    float *loss;
    int64_t *counts;
    float *w;
};
template <typename T, int N, int V, int L, int KL, int THREADS> void forward_launch(const Forward &f, hipStream_t s)
{
    balance_kernel<T, N, V, L, KL, THREADS><<<f.blocks, THREADS, 0, s>>>(
        static_cast<const T *>(f.scores), static_cast<const uint8_t *>(f.mask), f.Ttok, f.E, f.k, f.pp, f.pc, f.pn, f.loss,
        f.counts, f.w);
}
template <typename T, int N> void forward_sums(const Forward &f, hipStream_t s)
{
    if (f.k > kFewPicks) {
        if (f.E <= kFewExperts) forward_launch<T, N, 8, kPickLanesFew, 32, kPickThreads>(f, s);
        else forward_launch<T, N, 8, kPickLanesMany, 32, kPickThreads>(f, s);
    } else if (f.E <= kFewExperts) {
        switch (lanes_few(f.E)) {
            case 1: forward_launch<T, N, 8, 1, 8, kFewThreads>(f, s); break;
            case 2: forward_launch<T, N, 8, 2, 8, kFewThreads>(f, s); break;
            case 4: forward_launch<T, N, 8, 4, 8, kFewThreads>(f, s); break;
            default: forward_launch<T, N, 8, 8, 8, kFewThreads>(f, s); break;
        }
    } else if (lanes_many(f.E) == 8) {
        forward_launch<T, N, 16, 8, 8, kManyThreads>(f, s);
    } else {
        forward_launch<T, N, 16, 16, 8, kManyThreads>(f, s);
    }
}

// One block serves a decoding batch in one launch; beyond that at most one block per CU and a second launch.  With more
// picks a block holds fewer tokens at a time, and so there are more of them (4096 tokens, 100 experts, k = 9, fp32: 13 us; as many
// blocks as for few picks 52); for the tokens of a single block it takes up to 8 trips (64 tokens, 256 experts, k = 32: 22 us).
inline int blocks_for(int64_t Ttok, int E, int k)
{
    const bool few = E <= kFewExperts;
    const int64_t one = few ? kFewThreads / lanes_few(E) : kManyThreads / lanes_many(E);        // tokens of a block
    if (Ttok <= one) return 1;
    const int64_t b = ceil_div(Ttok, k <= kFewPicks ? one : kPickThreads / (few ? kPickLanesFew : kPickLanesMany));
    return static_cast<int>(b < kMaxBlocks ? b : kMaxBlocks);
}

template <typename T>
int forward_impl(const void *scores, const void *mask, int64_t Ttok, int E, int k, void *ws, float *loss, int64_t *counts,
                 float *w, hipStream_t s)
{
    constexpr int n = Vec16<T>::n;
    Forward f{scores, mask, Ttok, E, k, blocks_for(Ttok, E, k), static_cast<float *>(ws), nullptr, nullptr, loss, counts, w};
    f.pc = reinterpret_cast<int32_t *>(f.pp + f.blocks * pitch_of(E));
    f.pn = f.pc + f.blocks * pitch_of(E);
    if (E % n == 0 && aligned16(scores)) forward_sums<T, n>(f, s);
    else forward_sums<T, 1>(f, s);
    OPMX_LAUNCH_CHECK();
    if (f.blocks > 1) {
        balance_finish_kernel<<<1, kFinish, 0, s>>>(reinterpret_cast<const float4 *>(f.pp), reinterpret_cast<const int4 *>(f.pc), f.pn, f.blocks, E, k, loss, counts, w);
        OPMX_LAUNCH_CHECK();
    }
    return OPMX_OK;
}

struct Backward {
    const void *scores, *mask;
    const float *w, *dloss;
    int64_t Ttok;
    int E;
    void *dscores;
};
template <typename T, int N, int V, int L> void backward_launch(const Backward &b, hipStream_t s)
{
    const int64_t blocks = ceil_div(b.Ttok, 256 / L), most = 16 * 256;
    balance_backward_kernel<T, N, V, L><<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, s>>>(
        static_cast<const T *>(b.scores), static_cast<const uint8_t *>(b.mask), b.w, b.dloss, b.Ttok, b.E,
        static_cast<T *>(b.dscores));
}
template <typename T, int N> void backward_grads(const Backward &b, hipStream_t s)
{
    if (b.E <= kFewExperts) {
        switch (lanes_few(b.E)) {
            case 1: backward_launch<T, N, 8, 1>(b, s); break;
            case 2: backward_launch<T, N, 8, 2>(b, s); break;
            case 4: backward_launch<T, N, 8, 4>(b, s); break;
            default: backward_launch<T, N, 8, 8>(b, s); break;
        }
    } else if (lanes_many(b.E) == 8) {
        backward_launch<T, N, 16, 8>(b, s);
    } else {
        backward_launch<T, N, 16, 16>(b, s);
    }
}
template <typename T>
int backward_impl(const void *scores, const void *mask, const float *w, const float *dloss, int64_t Ttok, int E,
                  void *dscores, hipStream_t s)
{
    constexpr int n = Vec16<T>::n;
    const Backward b{scores, mask, w, dloss, Ttok, E, dscores};
    if (E % n == 0 && aligned16(scores) && aligned16(dscores)) backward_grads<T, n>(b, s);
    else backward_grads<T, 1>(b, s);
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

}  // namespace

size_t moe_balance_loss_workspace_bytes(int64_t Ttok, int E)
{
    if (Ttok <= 0 || E <= 0 || E > OPMX_MOE_MAX_EXPERTS) return 256;
    const int few = blocks_for(Ttok, E, kFewPicks), many = blocks_for(Ttok, E, kFewPicks + 1), blocks = few > many ? few : many;
    if (blocks == 1) return 256;             // finishes by itself
    const size_t b = static_cast<size_t>(blocks) * (static_cast<size_t>(pitch_of(E)) * 8 + 4);
    return (b + 255) / 256 * 256 + 256;
}

int launch_moe_balance_loss(const void *scores, const void *mask, int64_t T, int E, int k, int dtype, float *loss,
                            int64_t *counts, float *w, void *ws, hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return forward_impl<float>(scores, mask, T, E, k, ws, loss, counts, w, s);
        case OPMX_DTYPE_F16: return forward_impl<f16>(scores, mask, T, E, k, ws, loss, counts, w, s);
        case OPMX_DTYPE_BF16: return forward_impl<bf16>(scores, mask, T, E, k, ws, loss, counts, w, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

int launch_moe_balance_loss_backward(const void *scores, const void *mask, const float *w, const float *dloss, int64_t T,
                                     int E, int dtype, void *dscores, hipStream_t s)
{
    switch (dtype) {
        case OPMX_DTYPE_F32: return backward_impl<float>(scores, mask, w, dloss, T, E, dscores, s);
        case OPMX_DTYPE_F16: return backward_impl<f16>(scores, mask, w, dloss, T, E, dscores, s);
        case OPMX_DTYPE_BF16: return backward_impl<bf16>(scores, mask, w, dloss, T, E, dscores, s);
    }
    return OPMX_ERR_UNSUPPORTED;
}

}  // namespace opmx
