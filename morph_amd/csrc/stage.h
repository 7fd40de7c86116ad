// What the kernels of morph_state_space.h share: accesses of 16 bytes at any element, sums over waves.
#pragma once

#include "../../include/morph_state_space.h"
#include "layers.h"

namespace morph {

typedef uint32_t u32x4_half __attribute__((ext_vector_type(4), aligned(2)));

// 16 bytes of T at any element's address: gfx950 takes global accesses of 16 bytes at any address.
template <typename T>
struct Wide {
  static constexpr int kCount = 16 / Fmt<T>::bytes;
  typedef std::conditional_t<Fmt<T>::bytes == 4, u32x4_any, u32x4_half> raw;

  // The first n of kCount values (n >= kCount: all); the others are 0.
  static __device__ __forceinline__ u32x4 load(const void* p, int64_t at, int64_t n) {
    const char* q = static_cast<const char*>(p) + at * Fmt<T>::bytes;
    if (n >= kCount) return *reinterpret_cast<const raw*>(q);
    u32x4 w = 0;
#pragma unroll
    for (int k = 0; k < kCount; ++k)
      if (k < n) {
        if constexpr (Fmt<T>::bytes == 4) w[k] = reinterpret_cast<const uint32_t*>(q)[k];
        else w[k / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[k] << (16 * (k % 2));
      }
    return w;
  }
  static __device__ __forceinline__ void unpack(const u32x4& w, float (&x)[kCount]) {
#pragma unroll
    for (int k = 0; k < kCount; ++k) {
      if constexpr (Fmt<T>::bytes == 4) x[k] = __builtin_bit_cast(float, (uint32_t)w[k]);
      else x[k] = to_float<T>(k % 2 ? w[k / 2] >> 16 : w[k / 2] & 0xFFFFu);
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[kCount]) {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (Fmt<T>::bytes == 4) w[k] = __builtin_bit_cast(uint32_t, x[k]);
      else w[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
    }
    return w;
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const u32x4& w, int64_t n) {
    char* q = static_cast<char*>(p) + at * Fmt<T>::bytes;
    if (n >= kCount) {
      *reinterpret_cast<raw*>(q) = w;
      return;
    }
#pragma unroll
    for (int k = 0; k < kCount; ++k)
      if (k < n) {
        if constexpr (Fmt<T>::bytes == 4) reinterpret_cast<uint32_t*>(q)[k] = w[k];
        else reinterpret_cast<uint16_t*>(q)[k] = (uint16_t)(w[k / 2] >> (16 * (k % 2)));
      }
  }
};

template <typename T>
__device__ __forceinline__ float load_one(const void* p, int64_t i) {
  if constexpr (std::is_same_v<T, F32>) return static_cast<const float*>(p)[i];
  else return to_float<T>(static_cast<const uint16_t*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void store_one(void* p, int64_t i, float x) {
  if constexpr (std::is_same_v<T, F32>) static_cast<float*>(p)[i] = x;
  else static_cast<uint16_t*>(p)[i] = (uint16_t)pack2<T>(x, x);
}

// x from the lane that a DPP control names, within its row of 16 lanes.
template <int kControl>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kControl, 0xF, 0xF, true));
}
constexpr int kRotate1 = 0x121, kRotate2 = 0x122, kRotate4 = 0x124, kRotate8 = 0x128, kRotate12 = 0x12C;

// The sum over the wave, in every lane: rotations sum a row of 16 lanes, the swaps the four rows.
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<kRotate8>(x);
  x += dpp<kRotate4>(x);
  x += dpp<kRotate2>(x);
  x += dpp<kRotate1>(x);
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
}

inline bool known_dtype(int dtype) {
  return dtype == MORPH_DTYPE_F32 || dtype == MORPH_DTYPE_F16 || dtype == MORPH_DTYPE_BF16;
}

// f(T{}, W{}) for the activations' dtype and the weights' (F32 or the same).
template <typename F>
int by_dtypes(int dtype, int weight_dtype, F&& f) {
  const bool same = dtype == weight_dtype;
  if (!same && weight_dtype != MORPH_DTYPE_F32) return MORPH_EDTYPE;
  switch (dtype) {
    case MORPH_DTYPE_F32: return f(F32{}, F32{});
    case MORPH_DTYPE_F16: return same ? f(F16{}, F16{}) : f(F16{}, F32{});
    case MORPH_DTYPE_BF16: return same ? f(BF16{}, BF16{}) : f(BF16{}, F32{});
    default: return MORPH_EDTYPE;
  }
}

}  // namespace morph
