// Device mathematics that the layer operators share.
#pragma once

#include <type_traits>

#include "../../include/morph_layers.h"
#include "common.h"

namespace morph {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Whether so many workgroups of `threads` may be launched along a dimension: fewer than 2^32 threads.
inline bool launchable(int64_t workgroups, int64_t threads) {
  return workgroups <= int64_t(0xFFFFFFFF) / threads;
}

// Two floats in one word, each rounded to nearest even (overflow to inf, as a conversion).
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, F16>) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  }
}
// sigmoid(x) and sigmoid(-x) from one exponential of -|x|, which neither overflows nor
// cancels, so that the smaller one keeps its digits where 1 - sigmoid(x) would keep none.  The larger
// one is accurate to a few ulp.  The smaller one's relative error grows with |x|, since the product
// with log2(e) is rounded: up to 8 units of 2^-24 at |x| = 10, 16 at 20, 56 at 50 and 64 at 87
// (evaluated with an exact exponential).  +-inf give exactly 1 and 0, NaN gives NaN.
struct Sigmoid {
  float a, b;
};
__device__ __forceinline__ Sigmoid sigmoid(float x) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * __builtin_fabsf(x));
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  return x < 0.0f ? Sigmoid{small, big} : Sigmoid{big, small};
}

// sigmoid(x) alone, where 1 - sigmoid(x) is not needed or only added to: e^-x overflows to inf
// where it is 0.
__device__ __forceinline__ float gate_sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * x));
}

// silu(x) = x sigmoid(x) and its derivative.
struct Silu {
  float y, slope;
};
__device__ __forceinline__ Silu silu(float x) {
  const float a = gate_sigmoid(x), y = x * a;
  return Silu{y, __fmaf_rn(y, 1.0f - a, a)};
}

// ---- 8-bit activation groups (morph_layers.h) -------------------------------

// |x| as an integer that orders like it, and with 0 for inf and NaN: a group's scale comes
// from its finite values.
__device__ __forceinline__ uint32_t magnitude(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
  const uint32_t m = magnitude(x);
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
// not finite gets the NaN code (kFinite: there is none).
template <bool kFinite>
__device__ __forceinline__ uint32_t act_encode4(float x0, float x1, float x2, float x3,
                                                float inverse) {
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x0 * inverse, x1 * inverse, 0, false);
  w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2 * inverse, x3 * inverse, (int)w, true);
  if constexpr (!kFinite) {
    const float x[4] = {x0, x1, x2, x3};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (nonfinite_f32_bits(__builtin_bit_cast(uint32_t, x[k]))) w = (w & ~(0xFFu << (8 * k))) | (0x7Fu << (8 * k));
  }
  return w;
}
// The codes of kCount values of one lane and their group's exponent byte; most(m): the group's
// maximum of its lanes' m.  One test of the whole wave takes the form for finite values.
template <int kCount, typename Most>
__device__ __forceinline__ int act_encode(const float (&x)[kCount], uint32_t (&w)[kCount / 4], Most&& most) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < kCount; ++k) m = max(m, magnitude(x[k]));
  int e;
  if (__any(m >= 0x7F800000u)) {
    m = 0;
#pragma unroll
    for (int k = 0; k < kCount; ++k) m = max(m, finite_magnitude(x[k]));
    e = act_exponent(most(m));
#pragma unroll
    for (int k = 0; k < kCount; k += 4)
      w[k / 4] = act_encode4<false>(x[k], x[k + 1], x[k + 2], x[k + 3], act_inverse(e));
  } else {
    e = act_exponent(most(m));
#pragma unroll
    for (int k = 0; k < kCount; k += 4)
      w[k / 4] = act_encode4<true>(x[k], x[k + 1], x[k + 2], x[k + 3], act_inverse(e));
  }
  return e;
}
__device__ __forceinline__ void act_decode4(uint32_t w, float scale, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0] * scale;
  x[1] = lo[1] * scale;
  x[2] = hi[0] * scale;
  x[3] = hi[1] * scale;
}

// Values decoded for the type T, where an infinity (the code above the largest values) becomes T's largest
// value; NaN fails both comparisons.  Only groups of this exponent byte on hold such codes: 448 * 2^(e - 127)
// is in the range below it.
template <typename T>
constexpr int kActTop = std::is_same_v<T, F16> ? 135 : 247;
template <typename T, int kCount>
__device__ __forceinline__ void act_saturate(float (&x)[kCount]) {
  constexpr float kMost = std::is_same_v<T, F16> ? 65504.0f : std::is_same_v<T, BF16> ? 0x1.FEp127f : 0x1.FFFFFEp127f;
#pragma unroll
  for (int k = 0; k < kCount; ++k) x[k] = x[k] > kMost ? kMost : x[k] < -kMost ? -kMost : x[k];
}

// The largest value of a quad of lanes, in all four.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
  return x;
}

// ---- the gate of the feed-forward block --------------------------------------
// (An epilogue holds 256 values a lane with no other wave to fill in, so each instruction
// saved is microseconds a launch.)
__device__ __forceinline__ float ffn_gate(float g, float u) { return g * gate_sigmoid(g) * u; }

struct GateGrad {
  float h, dg, du;
};
__device__ __forceinline__ GateGrad ffn_gate_grad(float dh, float g, float u) {
  const Silu s = silu(g);
  return GateGrad{s.y * u, dh * u * s.slope, dh * s.y};
}

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x3_any __attribute__((ext_vector_type(3), aligned(4)));

// Eight values at any place, as they lie behind the 4-byte boundary at or before them (a value more in front, of
// the same allocation), and the last of them.
__device__ __forceinline__ u32x4 load_eight(const uint16_t* p) {
  const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 2) * 8, last = p[7];
  const u32x4 w = *reinterpret_cast<const u32x4_any*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
  return u32x4{__builtin_amdgcn_alignbit(w.y, w.x, shift), __builtin_amdgcn_alignbit(w.z, w.y, shift),
               __builtin_amdgcn_alignbit(w.w, w.z, shift), __builtin_amdgcn_alignbit(last, w.w, shift)};
}

// The first n of eight values to any place; vector: a multiple of 16 bytes.  At 2 mod 4 three
// stores, the middle one on 4-byte words (the weights' gradients of 3 rows of 2586 x 5905: 57 us, value by
// value 169).
__device__ __forceinline__ void store_eight(uint16_t* at, const u32x4 w, int64_t n, bool vector) {
  if (n >= 8) {
    if (vector) {
      *reinterpret_cast<u32x4*>(at) = w;
    } else if (reinterpret_cast<uintptr_t>(at) % 4 == 0) {
      *reinterpret_cast<u32x4_any*>(at) = w;
    } else {
      at[0] = (uint16_t)w.x;
      *reinterpret_cast<u32x3_any*>(at + 1) =
          u32x3_any{__builtin_amdgcn_alignbit(w.y, w.x, 16), __builtin_amdgcn_alignbit(w.z, w.y, 16),
                    __builtin_amdgcn_alignbit(w.w, w.z, 16)};
      at[7] = (uint16_t)(w.w >> 16);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) at[e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
  }
}

}  // namespace morph
