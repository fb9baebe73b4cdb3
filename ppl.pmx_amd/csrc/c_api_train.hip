// extern "C" surface of libopmx_moe.so, the operators for training: argument checks.  Declarations are in
// include/opmx_moe.h.
#include "train.h"

using namespace opmx;

namespace {

inline bool dtype_ok(int d) { return d == OPMX_DTYPE_F32 || d == OPMX_DTYPE_F16 || d == OPMX_DTYPE_BF16; }
inline size_t elt(int d) { return d == OPMX_DTYPE_F32 ? 4 : 2; }
inline hipStream_t st(void *s) { return static_cast<hipStream_t>(s); }

}  // namespace

extern "C" {

int opmx_checkpoint8_pack(const void *X, int64_t R, int64_t D, int dtype, int8_t *q, uint8_t *code, void *stream)
{
    if (R < 0 || D < 0) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype)) return OPMX_ERR_UNSUPPORTED;
    if (R == 0 || D == 0) return OPMX_OK;
    if (!X || !q || !code) return OPMX_ERR_BAD_ARGUMENT;
    return launch_checkpoint8_pack(X, R, D, dtype, q, code, st(stream));
}

int opmx_checkpoint8_unpack(const int8_t *q, const uint8_t *code, int64_t R, int64_t D, int dtype, void *X, void *stream)
{
    if (R < 0 || D < 0) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype)) return OPMX_ERR_UNSUPPORTED;
    if (R == 0 || D == 0) return OPMX_OK;
    if (!X || !q || !code) return OPMX_ERR_BAD_ARGUMENT;
    return launch_checkpoint8_unpack(q, code, R, D, dtype, X, st(stream));
}

int opmx_swiglu_checkpoint8(const void *X, int64_t R, int64_t D, float beta, int dtype, void *Y, int8_t *q, uint8_t *code,
                            void *stream)
{
    if (R < 0 || D < 0) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype)) return OPMX_ERR_UNSUPPORTED;
    if (R == 0 || D == 0) return OPMX_OK;
    if (!X || !Y || (q == nullptr) != (code == nullptr)) return OPMX_ERR_BAD_ARGUMENT;
    return launch_swiglu_checkpoint8(X, R, D, beta, dtype, Y, q, code, st(stream));
}

int opmx_swiglu_checkpoint8_backward(const void *dY, const int8_t *q, const uint8_t *code, int64_t R, int64_t D,
                                     float beta, int dtype, void *dX, void *stream)
{
    if (R < 0 || D < 0) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype)) return OPMX_ERR_UNSUPPORTED;
    if (R == 0 || D == 0) return OPMX_OK;
    if (!dY || !q || !code || !dX) return OPMX_ERR_BAD_ARGUMENT;
    return launch_swiglu_checkpoint8_backward(dY, q, code, R, D, beta, dtype, dX, st(stream));
}

// Sizes whose offsets inside a tile (256 rows) and whose counts of tiles and values stay in range.
static bool linear_sizes_ok(int64_t T, int64_t K, int64_t N)
{
    constexpr int64_t most = int64_t{1} << 21, rows = int64_t{1} << 31;
    return K < most && N < most && T < rows;
}

size_t opmx_linear_epilogue_kept_bytes(int64_t T, int64_t N, int dtype)
{
    if (T <= 0 || N <= 0 || !dtype_ok(dtype)) return 0;
    return static_cast<size_t>(T) * static_cast<size_t>(N) * (dtype == OPMX_DTYPE_F32 ? 4 : 3);
}

size_t opmx_linear_epilogue_workspace_bytes(int64_t T, int64_t K, int64_t N, int dtype, int activation)
{
    if (T <= 0 || K <= 0 || N <= 0 || !dtype_ok(dtype) || !linear_sizes_ok(T, K, N)) return 256;
    return linear_epilogue_workspace_bytes(T, K, N, dtype, activation);
}

int opmx_linear_epilogue(const void *X, const void *W, const void *B, const void *R, int64_t T, int64_t K, int64_t N,
                         int dtype, int activation, void *Y, void *H, void *workspace, size_t workspace_bytes, void *stream)
{
    if (T < 0 || K < 0 || N < 0 || activation < OPMX_ACTIVATION_NONE || activation > OPMX_ACTIVATION_SWIGLU)
        return OPMX_ERR_BAD_ARGUMENT;
    if (activation == OPMX_ACTIVATION_SWIGLU && N % 2) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype) || !linear_sizes_ok(T, K, N)) return OPMX_ERR_UNSUPPORTED;
    if (T == 0 || N == 0) return OPMX_OK;
    if (!X || !W || !Y || K == 0) return OPMX_ERR_BAD_ARGUMENT;
    if (K * static_cast<int64_t>(elt(dtype)) % 16 == 0 && !(aligned16(X) && aligned16(W))) return OPMX_ERR_ALIGNMENT;
    if (H && !aligned16(H)) return OPMX_ERR_ALIGNMENT;
    const size_t need = linear_epilogue_workspace_bytes(T, K, N, dtype, activation);
    if (need > 256 && (!workspace || workspace_bytes < need)) return OPMX_ERR_WORKSPACE;
    if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u)) return OPMX_ERR_ALIGNMENT;
    return launch_linear_epilogue(X, W, B, R, T, K, N, dtype, activation, Y, H, workspace, st(stream));
}

constexpr int kAnyGradients = OPMX_LINEAR_DX | OPMX_LINEAR_DW | OPMX_LINEAR_DB | OPMX_LINEAR_X8;

size_t opmx_linear_epilogue_backward_workspace_bytes(int64_t T, int64_t K, int64_t N, int dtype, int activation)
{
    if (T < 0 || K <= 0 || N <= 0 || !dtype_ok(dtype) || !linear_sizes_ok(T, K, N)) return 256;
    return linear_epilogue_backward_workspace_bytes(T, K, N, dtype, activation, kAnyGradients);
}

size_t opmx_linear_epilogue_gradients_workspace_bytes(int64_t T, int64_t K, int64_t N, int dtype, int activation, int wanted)
{
    if (T < 0 || K <= 0 || N <= 0 || !dtype_ok(dtype) || !linear_sizes_ok(T, K, N)) return 256;
    return linear_epilogue_backward_workspace_bytes(T, K, N, dtype, activation, T > 0 ? wanted : wanted & ~OPMX_LINEAR_DX);
}

// whatever: the workspace has to hold whatever may be asked for, not only what is.
static int linear_gradients(const void *dY, const void *X, const int8_t *x_q, const uint8_t *x_code, const void *W, const void *H,
                            int64_t T, int64_t K, int64_t N, int dtype, int activation, void *dX, void *dW, void *dB,
                            void *workspace, size_t workspace_bytes, void *stream, bool whatever)
{
    if (T < 0 || K < 0 || N < 0 || activation < OPMX_ACTIVATION_NONE || activation > OPMX_ACTIVATION_SWIGLU)
        return OPMX_ERR_BAD_ARGUMENT;
    if (activation == OPMX_ACTIVATION_SWIGLU && N % 2) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype) || !linear_sizes_ok(T, K, N)) return OPMX_ERR_UNSUPPORTED;
    if (K == 0 || N == 0) return OPMX_ERR_BAD_ARGUMENT;
    if (!dX && !dW && !dB) return OPMX_OK;
    if (T > 0) {
        if (!dY || (activation != OPMX_ACTIVATION_NONE && !H) || (dX && !W)) return OPMX_ERR_BAD_ARGUMENT;
        if (dW && !(x_q && x_code) && !X) return OPMX_ERR_BAD_ARGUMENT;
    }
    if ((x_q == nullptr) != (x_code == nullptr)) return OPMX_ERR_BAD_ARGUMENT;
    const int64_t size = static_cast<int64_t>(elt(dtype));
    if (K * size % 16 == 0 && ((dX && !aligned16(W)) || (dW && !x_q && !aligned16(X)))) return OPMX_ERR_ALIGNMENT;
    if (activation == OPMX_ACTIVATION_NONE && N * size % 16 == 0 && !aligned16(dY)) return OPMX_ERR_ALIGNMENT;
    if (H && !aligned16(H)) return OPMX_ERR_ALIGNMENT;
    if (T == 0) dX = nullptr;
    const int wanted = (dX ? OPMX_LINEAR_DX : 0) | (dW ? OPMX_LINEAR_DW : 0) | (dB ? OPMX_LINEAR_DB : 0) | (x_q ? OPMX_LINEAR_X8 : 0);
    const size_t need = linear_epilogue_backward_workspace_bytes(T, K, N, dtype, activation, whatever ? kAnyGradients : wanted);
    if (need > 256 && (!workspace || workspace_bytes < need)) return OPMX_ERR_WORKSPACE;
    if (workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u)) return OPMX_ERR_ALIGNMENT;
    return launch_linear_epilogue_backward(dY, X, x_q, x_code, W, H, T, K, N, dtype, activation, dX, dW, dB, wanted, workspace,
                                           st(stream));
}

int opmx_linear_epilogue_gradients(const void *dY, const void *X, const int8_t *x_q, const uint8_t *x_code, const void *W,
                                   const void *H, int64_t T, int64_t K, int64_t N, int dtype, int activation, void *dX,
                                   void *dW, void *dB, void *workspace, size_t workspace_bytes, void *stream)
{
    return linear_gradients(dY, X, x_q, x_code, W, H, T, K, N, dtype, activation, dX, dW, dB, workspace, workspace_bytes, stream,
                            false);
}

int opmx_linear_epilogue_backward(const void *dY, const void *X, const int8_t *x_q, const uint8_t *x_code, const void *W,
                                  const void *H, int64_t T, int64_t K, int64_t N, int dtype, int activation, void *dX,
                                  void *dW, void *dB, void *workspace, size_t workspace_bytes, void *stream)
{
    return linear_gradients(dY, X, x_q, x_code, W, H, T, K, N, dtype, activation, dX, dW, dB, workspace, workspace_bytes, stream,
                            true);
}

size_t opmx_moe_balance_loss_workspace_bytes(int64_t T, int E) { return moe_balance_loss_workspace_bytes(T, E); }

int opmx_moe_balance_loss(const void *scores, const uint8_t *token_mask, int64_t T, int E, int k, int dtype, float *loss,
                          int64_t *expert_count, float *weight, void *workspace, size_t workspace_bytes, void *stream)
{
    if (T < 0 || E <= 0 || k <= 0 || k > E) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype) || E > OPMX_MOE_MAX_EXPERTS || k > OPMX_MOE_MAX_EXPERTS_PER_TOKEN) return OPMX_ERR_UNSUPPORTED;
    if (T > ((int64_t{1} << 31) - 1) / k) return OPMX_ERR_UNSUPPORTED;        // counts of tokens are 32 bits on the way
    if (!loss || !expert_count || !weight || (T > 0 && !scores)) return OPMX_ERR_BAD_ARGUMENT;
    const size_t need = moe_balance_loss_workspace_bytes(T, E);
    if (need > 256 && (!workspace || workspace_bytes < need)) return OPMX_ERR_WORKSPACE;
    if (workspace && !aligned16(workspace)) return OPMX_ERR_ALIGNMENT;
    return launch_moe_balance_loss(scores, token_mask, T, E, k, dtype, loss, expert_count, weight, workspace, st(stream));
}

int opmx_moe_balance_loss_backward(const void *scores, const uint8_t *token_mask, const float *weight, const float *dloss,
                                   int64_t T, int E, int dtype, void *dscores, void *stream)
{
    if (T < 0 || E <= 0) return OPMX_ERR_BAD_ARGUMENT;
    if (!dtype_ok(dtype) || E > OPMX_MOE_MAX_EXPERTS) return OPMX_ERR_UNSUPPORTED;
    if (T == 0) return OPMX_OK;
    if (!scores || !weight || !dloss || !dscores) return OPMX_ERR_BAD_ARGUMENT;
    return launch_moe_balance_loss_backward(scores, token_mask, weight, dloss, T, E, dtype, dscores, st(stream));
}

}  // extern "C"
