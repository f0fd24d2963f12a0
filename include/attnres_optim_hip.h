/* attnres_optim_hip.h - C ABI of the optimizer step: AdamW over many tensors at once, as gfx950 HIP kernels.
 * Part of libattnres_hip.so.
 *
 * Contract, as in attnres_hip.h: device pointers (but for the table of tensors, which is read on the host before the
 * call returns); sizes in elements; the stream is passed explicitly (NULL: the legacy stream); the return value is 0 or
 * an attnres_status code, with a message from attnres_hip_last_error(); arguments are checked on the host before
 * anything is enqueued; no allocation, synchronisation, memset or host read of device memory, so a call can be captured
 * into a graph.  An element's result depends on nothing but its own values and, with 8-bit states, its block's.
 *
 * No counterpart in the reference, whose training step takes the optimizer from PyTorch (benchmarks/model.py:504-530).
 */
#ifndef ATTNRES_OPTIM_HIP_H
#define ATTNRES_OPTIM_HIP_H

#include <stdint.h>

#include "attnres_layers_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Elements that share a scale of 8-bit states: consecutive ones, counted from a tensor's first. */
#define ATTNRES_ADAMW_BLOCK 256

/* One tensor, its elements in one order in all of them and at their types' alignment.  With state_bits 32 exp_avg and
 * exp_avg_sq are FP32 and the scales NULL; with 8 they are E4M3 numbers (OCP: 3 bits of mantissa, largest 448),
 * one FP32 scale per ATTNRES_ADAMW_BLOCK of them: m = number * scale, and exp_avg_sq holds v's root.  master: FP32
 * weights of 16-bit parameters, or NULL. */
struct attnres_adamw_tensor {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* exp_avg_scale;
  float* exp_avg_sq_scale;
  float* master;
  int64_t elements;
};

/* One step, in place:
 *   g = grad * grad_scale;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g^2
 *   w = w (1 - lr weight_decay) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 * in FP32, w from master where there is one; param gets w rounded to its type.  8-bit states are rounded to nearest
 * after the step: numbers relative to the block's largest magnitude over 448, a root above zero never to zero.  A
 * gradient that is not finite makes its element NaN or infinite, and with 8-bit states its block's moments NaN.
 *
 * tensors: `count` of them in host memory, no two overlapping, of one param_dtype and one grad_dtype (param_dtype or
 * F32).  step (t >= 1) is read from step_device (int64) where that is not NULL, and lr from lr_device (FP32);
 * grad_scale: one FP32 value, or NULL for 1. */
int attnres_hip_adamw(const struct attnres_adamw_tensor* tensors, int64_t count, int param_dtype, int grad_dtype,
                      int state_bits, double lr, const float* lr_device, double beta1, double beta2, double eps,
                      double weight_decay, int64_t step, const int64_t* step_device, const float* grad_scale,
                      void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ATTNRES_OPTIM_HIP_H */
