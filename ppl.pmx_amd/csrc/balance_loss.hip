// Balance loss of the router and tokens per expert, with the gradient.
//
//   p[t, :] = softmax(scores[t, :]);  count[e] = kept tokens with e among their k largest scores;
//   f = count / (k n), n kept tokens;  loss = E sum_e f_e (1/n) sum_t p[t, e];
//   w_e = E f_e / n (held constant):  dscores[t, e] = dloss p[t, e] (w_e - sum_j w_j p[t, j]).
//
// The picks are MoeSelect's (ties to the lower expert id, NaN ranks first, -0 equals +0), so count is the
// difference of its expert_offset.  A row of -inf alone has p = 0: it has nothing to spread.
//
// Scores are read once in each direction and the gradient is written once.  A token belongs to L lanes
// (a power of two), each of which holds V of its E scores in registers.  A lane meets the same V experts in
// every token, so sums over tokens stay in registers until the block is done.  The k-th largest score
// comes from lists, not from k rounds of a wave-wide maximum: every lane keeps the KL largest of its keys sorted
// (one median-of-three per slot and key) and the lists of the L lanes meet in log2 L bitonic
// merges.  With E = 256, k = 8 that is about 45 vector instructions per token where the rounds take 600.
// An expert is picked where its key is not below the k-th; keys of 16-bit scores hold the id too and are
// distinct, equal fp32 scores at the k-th place are settled by id in a branch few waves take.
// Sums: fp32 in a lane (a few dozen tokens), 64 bits across blocks, in a fixed order: results do not vary.
#include "common.h"

namespace opmx {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / kWave;
constexpr int kMaxBlocks = 256;

template <typename T> struct Key {
    static constexpr bool unique = true;     // 16 bits of score, 16 bits of id
    static __device__ __forceinline__ uint32_t of(T v, int id)
    {
        uint16_t u;
        __builtin_memcpy(&u, &v, 2);
        const float f = to_f32(v);
        if (f != f) u = 0xFFFFu;
        else if (f == 0.0f) u = 0x8000u;
        else u = (u & 0x8000u) ? static_cast<uint16_t>(~u) : static_cast<uint16_t>(u | 0x8000u);
        return (static_cast<uint32_t>(u) << 16) | (0xFFFFu - static_cast<uint32_t>(id));
    }
};
template <> struct Key<float> {
    static constexpr bool unique = false;
    static __device__ __forceinline__ uint32_t of(float f, int)
    {
        if (f != f) return 0xFFFFFFFFu;
        const uint32_t u = __float_as_uint(f);
        if (f == 0.0f) return 0x80000000u;
        return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    }
};

__device__ __forceinline__ uint32_t umax_(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t umin_(uint32_t a, uint32_t b) { return a < b ? a : b; }

// The id of a lane's i-th score: chunks of N consecutive ids go round the L lanes of the token.
template <int N> __device__ __forceinline__ int expert_of(int i, int lane, int L) { return ((i / N) * L + lane) * N + i % N; }

// A lane's V scores of token t as floats; experts past E read as -inf.  keys (KEYS) get 0 there, which no
// score's key is.
template <typename T, int N, int V, bool KEYS>
__device__ __forceinline__ void load_scores(const T *__restrict__ row, int E, int lane, int L, float (&z)[V],
                                            uint32_t (&key)[KEYS ? V : 1])
{
#pragma unroll
    for (int c = 0; c < V / N; ++c) {
        const int e0 = (c * L + lane) * N;
        T v[N];
        const bool in = e0 < E;              // E % N == 0: a chunk is whole or absent
        if (in) {
            if constexpr (N == 1) v[0] = row[e0];
            else {
                const Vec16<T> q = load16_once(row + e0);
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = q.v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            z[c * N + j] = in ? to_f32(v[j]) : -INFINITY;
            if constexpr (KEYS) key[c * N + j] = in ? Key<T>::of(v[j], e0 + j) : 0u;
        }
    }
}

// z -> softmax over the token's L lanes.
template <int V> __device__ __forceinline__ void softmax_(float (&z)[V], int L)
{
    float m = z[0];
#pragma unroll
    for (int i = 1; i < V; ++i) m = fmaxf(m, z[i]);
    for (int d = 1; d < L; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
    const bool nothing = m == -INFINITY;     // (a NaN among the scores is not: it makes the sum NaN below)
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        z[i] = z[i] == -INFINITY ? 0.0f : expf(z[i] - m);
        sum += z[i];
    }
    for (int d = 1; d < L; d <<= 1) sum += __shfl_xor(sum, d, kWave);
    const float r = nothing && sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] *= r;
}

// Inserts x into the list a[0] >= a[1] >= ..., dropping the smallest.
template <int KL> __device__ __forceinline__ void insert(uint32_t (&a)[KL], uint32_t x)
{
#pragma unroll
    for (int j = KL - 1; j >= 1; --j)            // the median of x, a[j-1] >= a[j], in the form of v_med3_u32
        a[j] = umax_(umin_(x, a[j - 1]), umin_(umax_(x, a[j - 1]), a[j]));
    a[0] = umax_(a[0], x);
}

// a: the KL largest of a's and the xor-partner's lists, sorted again.
template <int KL> __device__ __forceinline__ void merge(uint32_t (&a)[KL], int d)
{
    uint32_t b[KL];
#pragma unroll
    for (int j = 0; j < KL; ++j) b[j] = __shfl_xor(a[KL - 1 - j], d, kWave);
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

template <int KL> __device__ __forceinline__ uint32_t at(const uint32_t (&a)[KL], int i)
{
    uint32_t v = a[0];
#pragma unroll
    for (int j = 1; j < KL; ++j) v = i == j ? a[j] : v;
    return v;
}

// What the sums over tokens become: loss, counts, and w for the backward pass.  One block.
__device__ __forceinline__ void finish(double psum, int64_t count, int64_t kept, int e, int E, int k, double *red,
                                       float *loss, int64_t *counts, float *w)
{
    const double n = kept > 0 ? static_cast<double>(kept) : 1.0;
    double part = 0.0;
    if (e < E) {
        const double f = static_cast<double>(count) / (static_cast<double>(k) * n);
        part = static_cast<double>(E) * f * (psum / n);
        counts[e] = count;
        w[e] = static_cast<float>(static_cast<double>(E) * f / n);
    }
    red[threadIdx.x] = part;
    __syncthreads();
    for (int s = kThreads / 2; s >= 1; s >>= 1) {
        if (static_cast<int>(threadIdx.x) < s) red[threadIdx.x] += red[threadIdx.x + s];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = static_cast<float>(red[0]);
}

// Sums over the tokens of a block.  A single block finishes by itself; several leave psum [blocks][E], counts
// [blocks][E] and kept [blocks] in the workspace.
template <typename T, int N, int V, int KL>
__global__ __launch_bounds__(kThreads) void balance_kernel(const T *__restrict__ scores,
                                                           const uint8_t *__restrict__ mask, int64_t Ttok, int E, int k,
                                                           int L, float *__restrict__ part_p, int32_t *__restrict__ part_c,
                                                           int32_t *__restrict__ part_n, float *__restrict__ loss,
                                                           int64_t *__restrict__ counts, float *__restrict__ w)
{
    __shared__ float s_p[kWaves][OPMX_MOE_MAX_EXPERTS];
    __shared__ int32_t s_c[kWaves][OPMX_MOE_MAX_EXPERTS];
    __shared__ int32_t s_n[kWaves];
    __shared__ double s_red[kThreads];
    const int lane = lane_id() % L, wave = threadIdx.x / kWave;
    const int per_block = kThreads / L;
    float psum[V];
    int32_t cnt[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        psum[i] = 0.0f;
        cnt[i] = 0;
    }
    int32_t kept = 0;
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * per_block; t0 < Ttok;
         t0 += static_cast<int64_t>(gridDim.x) * per_block) {
        const int64_t t = t0 + threadIdx.x / L;
        const bool keep = t < Ttok && (mask == nullptr || mask[t] != 0);     // the same in the token's L lanes
        const T *row = scores + (t < Ttok ? t : Ttok - 1) * E;
        float z[V];
        uint32_t key[V];
        load_scores<T, N, V, true>(row, E, lane, L, z, key);
        uint32_t list[KL];
#pragma unroll
        for (int j = 0; j < KL; ++j) list[j] = 0u;
#pragma unroll
        for (int i = 0; i < V; ++i) insert<KL>(list, key[i]);
        for (int d = 1; d < L; d <<= 1) merge<KL>(list, d);
        const uint32_t kth = at<KL>(list, k - 1);
        softmax_<V>(z, L);
        if constexpr (Key<T>::unique) {
#pragma unroll
            for (int i = 0; i < V; ++i) cnt[i] += keep && key[i] >= kth ? 1 : 0;
        } else {
            int above = 0, equal = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                above += key[i] > kth ? 1 : 0;
                equal += key[i] == kth ? 1 : 0;
            }
            for (int d = 1; d < L; d <<= 1) {
                above += __shfl_xor(above, d, kWave);
                equal += __shfl_xor(equal, d, kWave);
            }
            const int left = k - above;      // so many of the equal ones are picked, the lowest ids first
            if (!__any(equal > left)) {
#pragma unroll
                for (int i = 0; i < V; ++i) cnt[i] += keep && key[i] >= kth ? 1 : 0;
            } else {
                // ids go up chunk by chunk, and within a chunk lane by lane
                int before = 0;              // equal ones in the chunks behind us
#pragma unroll
                for (int c = 0; c < V / N; ++c) {
                    int mine = 0;
#pragma unroll
                    for (int j = 0; j < N; ++j) mine += key[c * N + j] == kth ? 1 : 0;
                    int upto = mine;
                    for (int d = 1; d < L; d <<= 1) {
                        const int o = __shfl_up(upto, d, kWave);
                        if (lane >= d) upto += o;
                    }
                    int rank = before + upto - mine;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const uint32_t q = key[c * N + j];
                        cnt[c * N + j] += keep && (q > kth || (q == kth && rank < left)) ? 1 : 0;
                        rank += q == kth ? 1 : 0;
                    }
                    before += __shfl(upto, (lane_id() / L) * L + L - 1, kWave);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) psum[i] += keep ? z[i] : 0.0f;
        kept += keep && lane == 0 ? 1 : 0;
    }
    // over the tokens of the wave, then of the block
#pragma unroll
    for (int i = 0; i < V; ++i) {
        for (int d = L; d < kWave; d <<= 1) {
            psum[i] += __shfl_xor(psum[i], d, kWave);
            cnt[i] += __shfl_xor(cnt[i], d, kWave);
        }
        const int e = expert_of<N>(i, lane, L);
        if (lane_id() < L && e < E) {
            s_p[wave][e] = psum[i];
            s_c[wave][e] = cnt[i];
        }
    }
    for (int d = 1; d < kWave; d <<= 1) kept += __shfl_xor(kept, d, kWave);
    if (lane_id() == 0) s_n[wave] = kept;
    __syncthreads();
    const int e = threadIdx.x;
    float p = 0.0f;
    int32_t c = 0, n = 0;
    if (e < E) {
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            p += s_p[v][e];
            c += s_c[v][e];
        }
    }
#pragma unroll
    for (int v = 0; v < kWaves; ++v) n += s_n[v];
    if (gridDim.x == 1) {
        finish(p, c, n, e, E, k, s_red, loss, counts, w);
        return;
    }
    if (e < E) {
        part_p[static_cast<int64_t>(blockIdx.x) * E + e] = p;
        part_c[static_cast<int64_t>(blockIdx.x) * E + e] = c;
    }
    if (e == 0) part_n[blockIdx.x] = n;
}

// The blocks' sums: thread (slice, e) adds every slices-th block's, in order, then slice 0 adds the slices.
__global__ __launch_bounds__(kThreads) void balance_finish_kernel(const float *__restrict__ part_p,
                                                                  const int32_t *__restrict__ part_c,
                                                                  const int32_t *__restrict__ part_n, int blocks, int E,
                                                                  int k, float *__restrict__ loss,
                                                                  int64_t *__restrict__ counts, float *__restrict__ w)
{
    __shared__ double s_red[kThreads];
    __shared__ int64_t s_c[kThreads];
    __shared__ int64_t s_n;
    const int slices = kThreads / E < 32 ? kThreads / E : 32;   // E <= 256: at least two
    const int slice = threadIdx.x / E, e = threadIdx.x % E;
    double p = 0.0;
    int64_t c = 0;
    if (slice < slices)
#pragma unroll 8
        for (int b = slice; b < blocks; b += slices) {
            p += part_p[b * E + e];
            c += part_c[b * E + e];
        }
    s_red[threadIdx.x] = p;
    s_c[threadIdx.x] = c;
    if (threadIdx.x < kWave) {
        int64_t n = 0;
        for (int b = threadIdx.x; b < blocks; b += kWave) n += part_n[b];
        for (int d = 1; d < kWave; d <<= 1) n += __shfl_xor(n, d, kWave);
        if (threadIdx.x == 0) s_n = n;
    }
    __syncthreads();
    if (slice == 0)
        for (int s = 1; s < slices; ++s) {
            p += s_red[s * E + e];
            c += s_c[s * E + e];
        }
    const int64_t n = s_n;
    __syncthreads();                         // s_red is used again
    finish(p, c, n, slice == 0 ? e : E, E, k, s_red, loss, counts, w);
}

template <typename T, int N, int V>
__global__ __launch_bounds__(256) void balance_backward_kernel(const T *__restrict__ scores,
                                                               const uint8_t *__restrict__ mask,
                                                               const float *__restrict__ w,
                                                               const float *__restrict__ dloss, int64_t Ttok, int E,
                                                               int L, T *__restrict__ dscores)
{
    const int lane = lane_id() % L, per_block = 256 / L;
    float wv[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = expert_of<N>(i, lane, L);
        wv[i] = e < E ? w[e] : 0.0f;
    }
    const float scale = *dloss;
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * per_block; t0 < Ttok;
         t0 += static_cast<int64_t>(gridDim.x) * per_block) {
        const int64_t t = t0 + threadIdx.x / L;
        const bool keep = t < Ttok && (mask == nullptr || mask[t] != 0);
        float z[V];
        uint32_t none[1];
        load_scores<T, N, V, false>(scores + (t < Ttok ? t : Ttok - 1) * E, E, lane, L, z, none);
        softmax_<V>(z, L);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) dot += z[i] * wv[i];
        for (int d = 1; d < L; d <<= 1) dot += __shfl_xor(dot, d, kWave);
        if (t >= Ttok) continue;             // (the last trip: nobody needs this lane again)
        T *out = dscores + t * E;
#pragma unroll
        for (int c = 0; c < V / N; ++c) {
            const int e0 = (c * L + lane) * N;
            if (e0 >= E) continue;
            T o[N];
#pragma unroll
            for (int j = 0; j < N; ++j)
                o[j] = from_f32<T>(keep ? scale * z[c * N + j] * (wv[c * N + j] - dot) : 0.0f);
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

// Lanes per token: E scores over V per lane.
inline int lanes_for(int E, int V, int N)
{
    int L = 1;
    while (L * V < (E + N - 1) / N * N) L <<= 1;
    return L;
}

// Up to 64 experts a lane holds 8 scores: more lanes per token, and the few tokens of a batch spread over more
// of them.  Beyond, 16: fewer merges per token, and registers for two waves per SIMD more than with 32.  Lists of 32 keys leave registers for 8 scores only.
constexpr int kFewExperts = 64;

template <typename T, int N, int V>
int balance_forward(const void *scores, const void *mask, int64_t Ttok, int E, int k, int blocks, float *pp, int32_t *pc,
                    int32_t *pn, float *loss, int64_t *counts, float *w, hipStream_t s)
{
    const int L = lanes_for(E, V, N);
    const T *z = static_cast<const T *>(scores);
    const uint8_t *m = static_cast<const uint8_t *>(mask);
    if (k <= 2) balance_kernel<T, N, V, 2><<<blocks, kThreads, 0, s>>>(z, m, Ttok, E, k, L, pp, pc, pn, loss, counts, w);
    else if (k <= 8) balance_kernel<T, N, V, 8><<<blocks, kThreads, 0, s>>>(z, m, Ttok, E, k, L, pp, pc, pn, loss, counts, w);
    else balance_kernel<T, N, 8, 32><<<blocks, kThreads, 0, s>>>(z, m, Ttok, E, k, lanes_for(E, 8, N), pp, pc, pn, loss,
                                                                counts, w);
    OPMX_LAUNCH_CHECK();
    if (blocks > 1) {
        balance_finish_kernel<<<1, kThreads, 0, s>>>(pp, pc, pn, blocks, E, k, loss, counts, w);
        OPMX_LAUNCH_CHECK();
    }
    return OPMX_OK;
}

template <typename T, int N, int V>
int balance_backward(const void *scores, const void *mask, const float *w, const float *dloss, int64_t Ttok, int E,
                     void *dscores, hipStream_t s)
{
    const int L = lanes_for(E, V, N);
    const int64_t blocks = ceil_div(Ttok, 256 / L), most = 16 * 256;
    balance_backward_kernel<T, N, V><<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, s>>>(
        static_cast<const T *>(scores), static_cast<const uint8_t *>(mask), w, dloss, Ttok, E, L, static_cast<T *>(dscores));
    OPMX_LAUNCH_CHECK();
    return OPMX_OK;
}

// One block serves a decoding batch in one launch; beyond that one block per CU and a second launch.
inline int blocks_for(int64_t Ttok, int E)
{
    const int L = lanes_for(E, E <= kFewExperts ? 8 : 16, 1);
    const int64_t b = ceil_div(Ttok, kThreads / L);
    return static_cast<int>(b <= 1 ? 1 : (b < kMaxBlocks ? b : kMaxBlocks));
}

template <typename T>
int forward_impl(const void *scores, const void *mask, int64_t Ttok, int E, int k, void *ws, float *loss, int64_t *counts,
                 float *w, hipStream_t s)
{
    constexpr int n = Vec16<T>::n;
    const int blocks = blocks_for(Ttok, E);
    float *pp = static_cast<float *>(ws);
    int32_t *pc = reinterpret_cast<int32_t *>(pp + static_cast<int64_t>(blocks) * E), *pn = pc + static_cast<int64_t>(blocks) * E;
    const bool vec = E % n == 0 && aligned16(scores);
    if (E <= kFewExperts)
        return vec ? balance_forward<T, n, 8>(scores, mask, Ttok, E, k, blocks, pp, pc, pn, loss, counts, w, s)
                   : balance_forward<T, 1, 8>(scores, mask, Ttok, E, k, blocks, pp, pc, pn, loss, counts, w, s);
    return vec ? balance_forward<T, n, 16>(scores, mask, Ttok, E, k, blocks, pp, pc, pn, loss, counts, w, s)
               : balance_forward<T, 1, 16>(scores, mask, Ttok, E, k, blocks, pp, pc, pn, loss, counts, w, s);
}

template <typename T>
int backward_impl(const void *scores, const void *mask, const float *w, const float *dloss, int64_t Ttok, int E,
                  void *dscores, hipStream_t s)
{
    constexpr int n = Vec16<T>::n;
    const bool vec = E % n == 0 && aligned16(scores) && aligned16(dscores);
    if (E <= kFewExperts)
        return vec ? balance_backward<T, n, 8>(scores, mask, w, dloss, Ttok, E, dscores, s)
                   : balance_backward<T, 1, 8>(scores, mask, w, dloss, Ttok, E, dscores, s);
    return vec ? balance_backward<T, n, 16>(scores, mask, w, dloss, Ttok, E, dscores, s)
               : balance_backward<T, 1, 16>(scores, mask, w, dloss, Ttok, E, dscores, s);
}

}  // namespace

size_t moe_balance_loss_workspace_bytes(int64_t Ttok, int E)
{
    if (Ttok <= 0 || E <= 0 || E > OPMX_MOE_MAX_EXPERTS) return 256;
    const size_t b = static_cast<size_t>(blocks_for(Ttok, E)) * (static_cast<size_t>(E) * 8 + 4);
    return (b + 255) / 256 * 256;
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
