/* attnres_layers_hip.h - C ABI of the layers around the residual reads:
 * layer norm, embedding and the softmax cross entropy over a vocabulary, each
 * forward and backward, as gfx950 HIP kernels.  Part of libattnres_hip.so.
 *
 * Contract, as in attnres_hip.h: device pointers; sizes and strides in
 * elements; the stream is passed explicitly (NULL: the legacy stream); the
 * return value is 0 or an attnres_status code, with a message from
 * attnres_hip_last_error(); arguments are checked on the host before anything
 * is enqueued; no allocation, synchronisation, memset or host read of device
 * memory, so every call can be captured into a graph; no state is shared
 * between calls, so calls with buffers of their own may overlap.  Results do not depend on
 * the order in which workgroups run: no floating-point atomics.
 *
 * These operators have no counterpart in the reference, whose model takes them
 * from PyTorch (benchmarks/model.py:180-355).
 */
#ifndef ATTNRES_LAYERS_HIP_H
#define ATTNRES_LAYERS_HIP_H

#include <stdint.h>

#include "attnres_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
enum attnres_dtype { ATTNRES_BF16 = 0, ATTNRES_F16 = 1, ATTNRES_F32 = 2 };

/* How a loss per token becomes the loss. */
enum attnres_reduction { ATTNRES_REDUCE_NONE = 0, ATTNRES_REDUCE_SUM = 1, ATTNRES_REDUCE_MEAN = 2 };

/* ---- layer norm ----
 * out = (x - mean) * rstd * weight + bias over rows [rows, width] of `dtype`,
 * 1 <= width <= ATTNRES_MAX_WIDTH, rows >= 0, mean and rstd = 1 / sqrt(var + eps)
 * in FP32.  x rows are x_stride apart; out is contiguous.  weight and bias [width]
 * are of param_dtype (dtype or F32), either may be NULL (ones; zeros).
 * stats: FP32 [2, rows] (mean, then rstd), or NULL when there is no backward. */
int attnres_hip_layer_norm_forward(const void* x, int64_t x_stride, int64_t rows, int64_t width, int dtype,
                                   const void* weight, const void* bias, int param_dtype, float eps, void* out,
                                   float* stats, void* stream);

/* FP32 elements of the backward's workspace (0 rows: 0; -1: outside the envelope). */
int64_t attnres_hip_layer_norm_workspace_elems(int64_t rows, int64_t width);

/* Gradients of the call above: grad_x contiguous [rows, width] of dtype, grad_weight
 * and grad_bias [width] of param_dtype; each may be NULL when it is not wanted.
 * grad_out rows are contiguous.  workspace: only with grad_weight or grad_bias. */
int attnres_hip_layer_norm_backward(const void* grad_out, const void* x, int64_t x_stride, int64_t rows, int64_t width,
                                    int dtype, const void* weight, int param_dtype, const float* stats, void* grad_x,
                                    void* grad_weight, void* grad_bias, float* workspace, int64_t workspace_elems,
                                    void* stream);

/* ---- embedding ----
 * out[b, t] = scale * weight[tokens[b, t]] + positions[t], rounded once to
 * out_dtype.  tokens [batch, length] contiguous, int64 (token_bytes 8) or int32
 * (4); weight [vocab, width] and positions [>= length, width] contiguous, of
 * weight_dtype; positions may be NULL.  A token outside 0..vocab-1 gives a row
 * of NaN and takes no part in the table's gradient. */
int attnres_hip_embedding_forward(const void* tokens, int token_bytes, int64_t batch, int64_t length,
                                  const void* weight, int64_t vocab, int64_t width, int weight_dtype,
                                  const void* positions, float scale, void* out, int out_dtype, void* stream);

/* Bytes of the backward's workspace (-1: outside the envelope), and of grad_positions alone (0: none needed). */
int64_t attnres_hip_embedding_workspace_bytes(int64_t batch, int64_t length, int64_t vocab, int64_t width);
int64_t attnres_hip_embedding_positions_workspace_bytes(int64_t batch, int64_t length, int64_t width);

/* Gradients: grad_weight [vocab, width] (every row written: zeros where no token
 * points) and grad_positions [position_rows, width] (zeros past length), of
 * weight_dtype; either may be NULL.  grad_out [batch, length, width] contiguous, of
 * out_dtype.  Rows are summed in FP32 in the order of the tokens.  Without grad_weight a workspace that is NULL or too small
 * is not used, and the sums over a large batch of few positions are not shared out (slower, other roundings). */
int attnres_hip_embedding_backward(const void* grad_out, int out_dtype, const void* tokens, int token_bytes,
                                   int64_t batch, int64_t length, int64_t vocab, int64_t width, int weight_dtype,
                                   float scale, void* grad_weight, void* grad_positions, int64_t position_rows,
                                   void* workspace, int64_t workspace_bytes, void* stream);

/* ---- softmax cross entropy of logits = hidden weight^T ----
 * hidden [rows, width] (rows hidden_stride apart), weight [vocab, width] (rows
 * weight_stride apart) of one dtype, 1 <= width <= ATTNRES_MAX_WIDTH, rows and vocab up
 * to 2^24 each and to 2^22 tiles of 256 x 256 together.  Where weight is of 16 bits and width a multiple of
 * 32, its rows start at multiples of 16 bytes, at most 2^22 elements apart (else ATTNRES_ERR_STRIDE): it is
 * multiplied where it lies.  targets [rows] contiguous, int64 or int32
 * (target_bytes).  loss (FP32): [rows] for ATTNRES_REDUCE_NONE (0 where the target
 * is ignore_index), else one value; the mean is over the targets that count (NaN
 * when none does).  A target that is neither ignore_index nor in 0..vocab-1 makes
 * the loss and the gradients NaN.
 * saved: what the backward reads.  keep, the same in all calls: nonzero lets the forward keep the exponentials of the
 * logits there for the backward, 2 bytes each for BF16 (and 4 per row, the target's logit), else 4, rows and vocab padded
 * to 256, where that takes at most 8 GiB, and its packed operands (of few rows, up to 64, the FP32 logits); otherwise, and with 0, saved is 256 + 20 * rows bytes and the backward
 * forms them again, for one piece of the vocabulary at a time.
 * workspace: backward 0 for the forward's, 1 for the backward's, 2 for that of a sum or a mean alone, which is smaller for F16 and
 * F32.  saved and workspace start at multiples of 16 bytes (else ATTNRES_ERR_WORKSPACE). */
int64_t attnres_hip_loss_saved_bytes(int64_t rows, int64_t vocab, int64_t width, int dtype, int keep);
int64_t attnres_hip_loss_workspace_bytes(int64_t rows, int64_t vocab, int64_t width, int dtype, int keep, int backward);

int attnres_hip_loss_forward(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                             const void* targets, int target_bytes, int64_t rows, int64_t vocab, int64_t width,
                             int dtype, int64_t ignore_index, int reduction, int keep, float* loss, void* saved,
                             void* workspace, int64_t workspace_bytes, void* stream);

/* grad_loss (FP32): one value, or [rows] for ATTNRES_REDUCE_NONE.  grad_hidden
 * [rows, width] and grad_weight [vocab, width] contiguous, of dtype; either may be NULL. */
int attnres_hip_loss_backward(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                              int64_t rows, int64_t vocab, int64_t width, int dtype, int reduction, int keep, const void* saved,
                              const float* grad_loss, void* grad_hidden, void* grad_weight, void* workspace,
                              int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ATTNRES_LAYERS_HIP_H */
