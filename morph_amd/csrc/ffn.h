// Library-internal parts of the gated feed-forward block: what one of its products reads and
// writes, and the epilogues that its kernels share.
#pragma once

#include <type_traits>

#include "layers.h"

namespace morph {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// A matrix operand: element (row, k) of a product's P or Q at p[row * rs + k * ks], one of
// the strides 1.  Rows run over M (P) or N (Q).
struct FfnOperand {
  const uint16_t* p;
  int64_t rs, ks;
};

// What a product does with its sums.
enum class FfnEpilogue {
  kStore,      // C = the sums
  kGate,       // P = x, Q[0] = gate, Q[1] = up: C = h = silu(g) * u, and g and u as `keep` says
  kGateGrad    // the sums are dh: C = h, dg and du from the g and u that were kept
};

// C [M, N] = sum over the segments of P[i] Q[i]^T over K each (kGate: one segment, and two
// products with the same P).  Internal buffers (h, dg, du, what is kept) have rows of
// `ld` = 32 G elements, zero behind ff; kStore writes rows of ldc.
struct FfnProduct {
  FfnOperand P[2], Q[2];
  int64_t M, N, K;
  int32_t segments;
  int32_t keep;
  uint16_t* C;
  int64_t ldc;
  uint16_t *dg, *du;
  void *g, *u;
  uint8_t *g_exponents, *u_exponents;
};

template <typename T>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same_v<T, F16>)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  return u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])};
}

// Keep eight consecutive values at index `at` of a row-major buffer whose rows are whole
// groups: FP32, or codes and the group's exponent, of which a quad of lanes holds four parts.
__device__ __forceinline__ void ffn_keep8(int keep, void* buffer, uint8_t* exponents, int64_t at,
                                          const float (&x)[8]) {
  if (keep == MORPH_FFN_KEEP_FULL) {
    float* p = static_cast<float*>(buffer) + at;
    *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else if (keep == MORPH_FFN_KEEP_ACT8) {
    uint32_t w[2];
    const int e = act_encode<8>(x, w, [](uint32_t m) { return quad_max(m); });
    *reinterpret_cast<u32x2*>(static_cast<uint8_t*>(buffer) + at) = u32x2{w[0], w[1]};
    if (at % MORPH_ACT_GROUP == 0) exponents[at / MORPH_ACT_GROUP] = (uint8_t)e;
  }
}

__device__ __forceinline__ void ffn_kept8(int keep, const void* buffer, const uint8_t* exponents,
                                          int64_t at, float (&x)[8]) {
  if (keep == MORPH_FFN_KEEP_FULL) {
    const float* p = static_cast<const float*>(buffer) + at;
    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = lo[k], x[4 + k] = hi[k];
  } else {
    const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(buffer) + at);
    const float scale = act_scale(exponents[at / MORPH_ACT_GROUP]);
    float lo[4], hi[4];
    act_decode4(w.x, scale, lo);
    act_decode4(w.y, scale, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = lo[k], x[4 + k] = hi[k];
  }
}

}  // namespace morph
