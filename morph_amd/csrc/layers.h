// Device mathematics that the layer operators share.
#pragma once

#include "../../include/morph_layers.h"
#include "common.h"

namespace morph {

// sigmoid(x) and sigmoid(-x) from one exponential of -|x|, which neither overflows nor
// cancels: both are accurate to a few ulp at either end, where 1 - sigmoid(x) would keep no
// digit.  +-inf give exactly 1 and 0, NaN gives NaN.
struct Sigmoid {
  float a, b;
};
__device__ __forceinline__ Sigmoid sigmoid(float x) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * __builtin_fabsf(x));
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  return x < 0.0f ? Sigmoid{small, big} : Sigmoid{big, small};
}

// ---- 8-bit activation groups (morph_layers.h) -------------------------------

// |x| as an integer that orders like it, with 0 for inf and NaN: the group's scale comes
// from its finite values.
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t m = __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu;
  return m < 0x7F800000u ? m : 0u;
}
// The exponent byte of a group whose largest finite magnitude has these bits: with
// amax = m 2^E, 1 <= m < 2, and 448 = 1.75 2^8, the least k with amax <= 448 2^k is E - 8, one
// more where m > 1.75.  The sum carries into the exponent field exactly then.
__device__ __forceinline__ int act_exponent(uint32_t amax_bits) {
  const int e = (int)((amax_bits + 0x1FFFFFu) >> 23) - 8;
  return e < 1 ? 1 : e;  // 247 at most: the largest finite float
}
__device__ __forceinline__ float act_scale(int e) {  // 2^(e - 127)
  return __builtin_bit_cast(float, (uint32_t)e << 23);
}
__device__ __forceinline__ float act_inverse(int e) {  // 2^(127 - e), e <= 253
  return __builtin_bit_cast(float, (uint32_t)(254 - e) << 23);
}
// Four codes of one word.  The multiplication is exact but where the product is subnormal,
// far below half of the least code.  gfx950's conversion rounds to nearest even; what is
// not finite gets the NaN code.
__device__ __forceinline__ uint32_t act_encode4(float x0, float x1, float x2, float x3,
                                                float inverse) {
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x0 * inverse, x1 * inverse, 0, false);
  w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2 * inverse, x3 * inverse, (int)w, true);
  const float x[4] = {x0, x1, x2, x3};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (nonfinite_f32_bits(__builtin_bit_cast(uint32_t, x[k]))) w = (w & ~(0xFFu << (8 * k))) | (0x7Fu << (8 * k));
  return w;
}
__device__ __forceinline__ void act_decode4(uint32_t w, float scale, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0] * scale;
  x[1] = lo[1] * scale;
  x[2] = hi[0] * scale;
  x[3] = hi[1] * scale;
}

// The largest value of a quad of lanes, in all four.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
  return x;
}

// ---- the gate of the feed-forward block --------------------------------------
__device__ __forceinline__ float ffn_gate(float g, float u) { return g * sigmoid(g).a * u; }

struct GateGrad {
  float h, dg, du;
};
__device__ __forceinline__ GateGrad ffn_gate_grad(float dh, float g, float u) {
  const Sigmoid s = sigmoid(g);
  const float act = g * s.a;
  return GateGrad{act * u, dh * u * (s.a * __fmaf_rn(g, s.b, 1.0f)), dh * act};
}

}  // namespace morph
