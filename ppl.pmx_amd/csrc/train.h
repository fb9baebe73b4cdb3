// Launch entry points of the operators for training (opmx_moe.h).  Apart from common.h, which is part of the layer's sources.
#pragma once
#include "common.h"

namespace opmx {

// 8-bit activation checkpoints (checkpoint8.h): q [R,D] whole numbers, codes [R, ceil(D/32)] (SwiGLU: both halves
// of a row on their own, q [R,2,D], codes [R,2,ceil(D/32)]).
int launch_checkpoint8_pack(const void *X, int64_t R, int64_t D, int dtype, void *q, void *codes, hipStream_t s);
// pitch: values from one row of X to the next (0: D)
int launch_checkpoint8_unpack(const void *q, const void *codes, int64_t R, int64_t D, int dtype, void *X, hipStream_t s,
                              int64_t pitch = 0);
int launch_swiglu_checkpoint8(const void *X, int64_t R, int64_t D, float beta, int dtype, void *Y, void *q, void *codes,
                              hipStream_t s);
int launch_swiglu_checkpoint8_backward(const void *dY, const void *q, const void *codes, int64_t R, int64_t D, float beta,
                                       int dtype, void *dX, hipStream_t s);
size_t linear_epilogue_workspace_bytes(int64_t T, int64_t K, int64_t N, int dtype, int act);
// wanted: opmx_linear_gradient
size_t linear_epilogue_backward_workspace_bytes(int64_t T, int64_t K, int64_t N, int dtype, int act, int wanted);
int launch_linear_epilogue(const void *X, const void *W, const void *B, const void *R, int64_t T, int64_t K, int64_t N,
                           int dtype, int act, void *Y, void *H, void *ws, hipStream_t s);
int launch_linear_epilogue_backward(const void *dY, const void *X, const void *xq, const void *xcode, const void *W,
                                    const void *H, int64_t T, int64_t K, int64_t N, int dtype, int act, void *dX, void *dW,
                                    void *dB, int wanted, void *ws, hipStream_t s);
size_t moe_balance_loss_workspace_bytes(int64_t T, int E);
int launch_moe_balance_loss(const void *scores, const void *mask, int64_t T, int E, int k, int dtype, float *loss,
                            int64_t *counts, float *w, void *ws, hipStream_t s);
int launch_moe_balance_loss_backward(const void *scores, const void *mask, const float *w, const float *dloss, int64_t T,
                                     int E, int dtype, void *dscores, hipStream_t s);

}  // namespace opmx
