/*
 * morph_state_space.h -- C ABI of the operators of a state space stage on MI355X (gfx950), beside the layer
 * operators of morph_layers.h.
 *
 *   layer norm                            morph_norm_forward, morph_norm_backward
 *   short causal convolution              morph_conv_forward, morph_conv_backward
 *   selective state space scan            morph_ssm_forward, morph_ssm_backward
 *
 * The conventions are morph_layers.h's.  Activations are F32, F16 or BF16 (`dtype`), all sums, states and
 * statistics FP32.  Weights are FP32, or where a weight dtype is given of that type, FP32 or the
 * activations'; their gradients have the weights' type.
 */
#ifndef MORPH_STATE_SPACE_H
#define MORPH_STATE_SPACE_H

#include "morph_optim.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Layer norm ------------------------------------------------------------
 *   xh = (x - mean) r, r = 1 / sqrt(mean((x - mean)^2) + eps), y = xh weight + bias
 * along each row of x [rows, cols].  Without weight: 1; without bias: 0.
 *
 * Backward, with g = dy weight: dx = r (g - mean(g) - xh mean(g xh)),
 * dweight = sum over rows of dy xh, dbias = sum over rows of dy.
 */
typedef struct morph_norm {
  const void* x;      /* [rows, cols], row stride x_ld */
  const void* weight; /* [cols] or NULL */
  const void* bias;   /* [cols] or NULL */
  int64_t rows, cols, x_ld;
  float eps;
  int32_t weight_dtype; /* of weight and bias: F32 or dtype */
} morph_norm;

/* y: [rows, cols], contiguous.  stats (NULL: not): float [2, rows], each row's mean and r. */
int morph_norm_forward(const morph_norm* norm, int dtype, void* y, float* stats, void* stream);
/* Bytes of the backward's workspace (16-byte aligned, any contents). */
size_t morph_norm_workspace_bytes(int64_t rows, int64_t cols);
/* dx: [rows, cols] contiguous.  dweight, dbias: [cols], or NULL. */
int morph_norm_backward(const morph_norm* norm, int dtype, const float* stats, const void* dy,
                        int64_t dy_ld, void* dx, void* dweight, void* dbias, void* workspace,
                        size_t workspace_bytes, void* stream);

/* ---- Short causal convolution ----------------------------------------------
 *   p_t = bias + sum over k of weight_k x_(t - taps + 1 + k),  y_t = p_t sigmoid(p_t)
 * for x [batch, steps, dim], every channel on its own; x before the first step is `before` [batch, taps - 1,
 * dim] (NULL: zeros), `after` the last taps - 1 inputs of before and x.
 *
 * Backward: dp = dy silu'(p), dx_t = sum over k of weight_k dp_(t + taps - 1 - k), with dafter added where x
 * is part of `after`; dweight_k = sum of dp_t x_(t - taps + 1 + k), dbias = sum of dp.
 */
#define MORPH_CONV_MAX_TAPS 4

typedef struct morph_conv {
  const void* x;
  const void* before;
  const void* weight; /* [dim, taps] contiguous, weight_dtype */
  const void* bias;   /* [dim] or NULL */
  int64_t batch, steps, dim;
  int64_t x_batch, x_step; /* strides; before and after are contiguous */
  int32_t taps;            /* 2 .. MORPH_CONV_MAX_TAPS */
  int32_t weight_dtype;    /* F32 or dtype */
} morph_conv;

/* y: [batch, steps, dim] contiguous; after: [batch, taps - 1, dim]. */
int morph_conv_forward(const morph_conv* conv, int dtype, void* y, void* after, void* stream);
size_t morph_conv_workspace_bytes(int64_t batch, int64_t steps, int64_t dim, int taps);
/* dx: contiguous; dweight: [dim, taps], dbias: [dim] or NULL; dbefore: as before, or NULL; dafter: NULL for
 * zeros. */
int morph_conv_backward(const morph_conv* conv, int dtype, const void* dy, int64_t dy_batch,
                        int64_t dy_step, const void* dafter, void* dx, void* dweight, void* dbias,
                        void* dbefore, void* workspace, size_t workspace_bytes, void* stream);

/* ---- Selective state space scan --------------------------------------------
 *   d_t = softplus(dt_t + dt_bias), h_t = exp(d_t A) h_(t-1) + d_t x_t B_t,
 *   y_t = (sum over n of C_t h_t + skip x_t) silu(z_t)
 * for x, dt, z [batch, steps, dim], B and C [batch, steps, states], A [dim, states], states h [batch, dim,
 * states] in FP32.  Without z, skip, dt_bias, first state: 1, 0, 0, 0.  dt = -inf passes a state on unchanged
 * (padding, with x, B and C finite).  A positive A is taken while exp(A times the sum of d over the steps) stays
 * finite: products of gates over many steps are formed.
 *
 * Backward, with ds = dy silu(z): r_t = ds_t C_t + exp(d_(t+1) A) r_(t+1), with dlast added to the last;
 *   dx = d sum_n(r B) + skip ds, dB = sum over channels of r d x, dC = sum over channels of h ds,
 *   dd = x sum_n(r B) + sum_n(w A), dA = sum of w d, w = r_t exp(d_t A) h_(t-1),
 *   ddt = dd sigmoid(dt + dt_bias), ddt_bias = sum of ddt, dskip = sum of ds x, dz = dy s silu'(z),
 *   dfirst = exp(d_1 A) r_1.
 *
 * kept: float [batch, ceil(steps / MORPH_SSM_SPAN), dim, states], the state that each span of steps begins
 * with; written by the forward (NULL: not), read by the backward.
 */
#define MORPH_SSM_SPAN 32
#define MORPH_SSM_MAX_STATES 64
#define MORPH_SSM_MAX_STEP (1 << 25) /* of dim, and of the step strides in elements */

typedef struct morph_ssm {
  const void* x;
  const void* dt;
  const void* z;        /* NULL: no output gate */
  const void* B;
  const void* C;
  const float* A;       /* [dim, states] contiguous */
  const float* skip;    /* [dim] or NULL */
  const float* dt_bias; /* [dim] or NULL */
  const float* first;   /* [batch, dim, states] or NULL */
  int64_t batch, steps, dim;
  int64_t x_batch, x_step, dt_batch, dt_step, z_batch, z_step, B_batch, B_step, C_batch, C_step;
  int32_t states;       /* 1 .. MORPH_SSM_MAX_STATES */
  int32_t reserved;     /* 0 */
} morph_ssm;

/* Bytes of the workspace (16-byte aligned, any contents) of a forward (backward = 0) or backward; may be 0. */
size_t morph_ssm_workspace_bytes(int64_t batch, int64_t steps, int64_t dim, int states, int backward);
/* y: [batch, steps, dim] contiguous; last: [batch, dim, states]. */
int morph_ssm_forward(const morph_ssm* ssm, int dtype, void* y, float* last, float* kept, void* workspace,
                      size_t workspace_bytes, void* stream);

/* What a backward writes, all contiguous; NULL only where the forward had none of it (dz, dskip,
 * ddt_bias) and for dfirst. */
typedef struct morph_ssm_grads {
  void* dx;
  void* ddt;
  void* dz;
  void* dB;
  void* dC;
  float* dA;
  float* dskip;
  float* ddt_bias;
  float* dfirst;
} morph_ssm_grads;

/* dlast: NULL for zeros. */
int morph_ssm_backward(const morph_ssm* ssm, int dtype, const float* kept, const void* dy,
                       int64_t dy_batch, int64_t dy_step, const float* dlast,
                       const morph_ssm_grads* grads, void* workspace, size_t workspace_bytes,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MORPH_STATE_SPACE_H */
