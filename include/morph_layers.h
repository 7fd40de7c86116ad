/*
 * morph_layers.h -- C ABI of the layer operators on MI355X (gfx950): what a streamed
 * stage computes between the weights that it loads and the gradients that it hands to
 * the optimizer step of morph_optim.h.
 *
 *   activation checkpoints in 8 bits      morph_act_pack, morph_act_unpack
 *   gated feed-forward block              morph_ffn_forward, morph_ffn_backward
 *   gated linear recurrence               morph_scan_forward, morph_scan_backward
 *
 * The conventions are morph_optim.h's: device pointers owned by the caller, no device
 * memory allocated and no state kept between calls, work enqueued on `stream`, 0 or a
 * negative MORPH_E* code returned, and then nothing enqueued.  Leading dimensions and
 * strides count elements.  Outputs may not overlap inputs.
 */
#ifndef MORPH_LAYERS_H
#define MORPH_LAYERS_H

#include "morph_optim.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Activation checkpoints in 8 bits --------------------------------------
 * A row of `cols` values is held as G = ceil(cols / 32) groups of 32 consecutive ones:
 * E4M3 codes [rows, 32 G] (zeros behind the last value) and one exponent byte per
 * group [rows, G].  With amax the largest finite magnitude of a group, its byte e is
 * the least value of 1 .. 247 with amax <= 448 * 2^(e - 127); a code is the value
 * times 2^(127 - e), rounded to the nearest E4M3 value (ties to even).  A value that is
 * not finite gets the NaN code and leaves the others of its group as they are: it
 * reaches the gradients as NaN, where the step's detector finds it.
 */
#define MORPH_ACT_GROUP 32

/* src: [rows, cols] of dtype F32, F16 or BF16, row stride ld >= cols. */
int morph_act_pack(const void* src, int dtype, int64_t rows, int64_t cols, int64_t ld,
                   uint8_t* codes, uint8_t* exponents, void* stream);
/* dst: [rows, cols] = dtype(code * 2^(e - 127)), row stride ld >= cols.  The nearest code may stand
 * for more than the value did: 63488 and above become 65536, as 1.9375 * 2^127 and above become 2^128.
 * In F16, and in F32 and BF16, that is infinite.  With MORPH_ACT_SATURATE added to dtype it becomes the
 * dtype's largest value, so that what was finite in this dtype comes back finite; NaN stays NaN. */
#define MORPH_ACT_SATURATE 0x100
int morph_act_unpack(const uint8_t* codes, const uint8_t* exponents, int64_t rows, int64_t cols,
                     void* dst, int dtype, int64_t ld, void* stream);

/* ---- Gated feed-forward block ----------------------------------------------
 *   g = x gate^T, u = x up^T, h = silu(g) * u, y = h down^T,  silu(g) = g / (1 + e^-g)
 * for x [rows, d], gate and up [ff, d], down [d, ff], all F16 or all BF16.  Sums are in
 * FP32; h is rounded to the element type (the matrix instructions read 16 bits).
 *
 * Backward, from dy [rows, d] and what the forward kept of g, u and x:
 *   dh = dy down, dg = dh u s (1 + g (1 - s)), du = dh g s,  s = 1 / (1 + e^-g)
 *   dx = dg gate + du up, dgate = dg^T x, dup = du^T x, ddown = dy^T h
 * dg, du and h are rounded to the element type, each gradient once at its end.
 */
enum morph_ffn_keep {
  MORPH_FFN_KEEP_NONE = 0, /* nothing: no backward follows */
  MORPH_FFN_KEEP_FULL = 1, /* g and u in FP32, and the caller keeps x */
  MORPH_FFN_KEEP_ACT8 = 2  /* g, u and x in 8 bits (the groups above); the backward decodes x with
                              MORPH_ACT_SATURATE, g and u in FP32 (infinite from 1.9375 * 2^127 on) */
};

typedef struct morph_ffn {
  const void* x;    /* [rows, d], row stride x_ld */
  const void* gate; /* [ff, d], row stride gate_ld */
  const void* up;   /* [ff, d], row stride up_ld */
  const void* down; /* [d, ff], row stride down_ld */
  int64_t rows, d, ff;
  int64_t x_ld, gate_ld, up_ld, down_ld;
} morph_ffn;

/* What lies between forward and backward, G = ceil(ff / 32), GX = ceil(d / 32).
 * FULL: gate and up are float [rows, 32 G].  ACT8: they are codes [rows, 32 G] with
 * exponents [rows, G]; x_codes [rows, 32 GX], x_exponents [rows, GX].  All 16-byte aligned. */
typedef struct morph_ffn_saved {
  int32_t keep; /* enum morph_ffn_keep */
  int32_t reserved;
  void* gate;
  void* up;
  uint8_t* gate_exponents;
  uint8_t* up_exponents;
  uint8_t* x_codes;
  uint8_t* x_exponents;
} morph_ffn_saved;

/* Bytes of workspace (16-byte aligned, any contents) of a forward (backward = 0) or backward. */
size_t morph_ffn_workspace_bytes(int64_t rows, int64_t d, int64_t ff, int keep, int backward);
/* y: [rows, d], row stride y_ld.  saved: NULL for MORPH_FFN_KEEP_NONE. */
int morph_ffn_forward(const morph_ffn* block, int dtype, const morph_ffn_saved* saved, void* y,
                      int64_t y_ld, void* workspace, size_t workspace_bytes, void* stream);
/* dx: [rows, d], dgate and dup: [ff, d], ddown: [d, ff], contiguous, each written whole.
 * block->x is read with MORPH_FFN_KEEP_FULL only. */
int morph_ffn_backward(const morph_ffn* block, int dtype, const morph_ffn_saved* saved,
                       const void* dy, int64_t dy_ld, void* dx, void* dgate, void* dup,
                       void* ddown, void* workspace, size_t workspace_bytes, void* stream);

/* ---- Gated linear recurrence -----------------------------------------------
 *   a_t = sigmoid(f_t), s_t = a_t s_(t-1) + (1 - a_t) v_t, y_t = s_t silu(z_t)
 * for f, v, z [batch, steps, dim] of one dtype (F32, F16 or BF16), dim contiguous; without
 * z, y_t = s_t.  f = -inf forgets a finite state exactly, +inf passes it on unchanged.  States
 * are FP32 throughout: s0 [batch, dim] (NULL: zeros), last [batch, dim] = s_steps.
 *
 * Backward, from dy and the gradient of the last state (NULL: zeros):
 *   r_t = dy_t silu(z_t) + a_(t+1) r_(t+1), with dlast added to the last
 *   dv_t = (1 - a_t) r_t, df_t = r_t (s_(t-1) - v_t) a_t (1 - a_t),
 *   dz_t = dy_t s_t silu'(z_t), ds0 = a_1 r_1
 *
 * states: FP32 [batch, ceil(steps / MORPH_SCAN_SPAN), dim], the state that each span
 * of steps begins with; written by the forward (NULL: not), read by the backward.
 */
#define MORPH_SCAN_SPAN 64

typedef struct morph_scan {
  const void* f;
  const void* v;
  const void* z; /* NULL: no output gate */
  const float* s0;
  int64_t batch, steps, dim;
  int64_t f_batch, f_step, v_batch, v_step, z_batch, z_step; /* strides */
} morph_scan;

/* Bytes of workspace (16-byte aligned, any contents); may be 0. */
size_t morph_scan_workspace_bytes(int64_t batch, int64_t steps, int64_t dim, int dtype, int backward);
/* y: [batch, steps, dim] contiguous. */
int morph_scan_forward(const morph_scan* scan, int dtype, void* y, float* last, float* states,
                       void* workspace, size_t workspace_bytes, void* stream);
/* dy: strides dy_batch, dy_step; df, dv, dz (with z): contiguous; ds0: [batch, dim]. */
int morph_scan_backward(const morph_scan* scan, int dtype, const float* states, const void* dy,
                        int64_t dy_batch, int64_t dy_step, const float* dlast, void* df, void* dv,
                        void* dz, float* ds0, void* workspace, size_t workspace_bytes,
                        void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MORPH_LAYERS_H */
