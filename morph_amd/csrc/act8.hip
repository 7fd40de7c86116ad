// Activation checkpoints in 8 bits (morph_layers.h): E4M3 codes with a power-of-two scale
// per 32 consecutive values of a row.
//
// A power of two as scale keeps the division and the multiplication back exact, so a value
// is rounded once, and one byte holds it; a floating code loses nothing by it but where a
// group spans more than E4M3's 2^17.  32 values are what the feed-forward block's epilogue
// holds of a row in one wave (ffn kernels), so the same groups are written there without a
// pass of their own.
//
// Four lanes hold a group, eight values each: the maximum is a reduction within a quad
// (two DPP steps), and a wave reads whole lines and writes 512 contiguous codes.
#include <type_traits>

#include "layers.h"

namespace morph {
namespace {

constexpr int kGroup = MORPH_ACT_GROUP;
constexpr int kThreads = 256;
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Values c .. c + 7 of a row of `cols` (zeros behind its end); wide: the row's address and
// stride allow 16-byte accesses.  Others go by words: 11308 x 2763 in BF16, pack and unpack, 39 us (value by
// value 85), 2762 in FP32 59 (140).
template <typename T>
__device__ __forceinline__ void load8(const void* row, int64_t c, int64_t cols, bool wide,
                                      float (&x)[8]) {
  if constexpr (std::is_same_v<T, F32>) {
    const float* p = static_cast<const float*>(row) + c;
    if (c + 8 <= cols) {
      const f32x4 lo = *reinterpret_cast<const f32x4_any*>(p), hi = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = lo[k], x[4 + k] = hi[k];
      return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = c + k < cols ? p[k] : 0.0f;
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(row) + c;
    if (c + 8 <= cols) {
      const u32x4 v = wide ? *reinterpret_cast<const u32x4*>(p) : load_eight(p);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[2 * k] = to_float<T>(v[k] & 0xFFFFu);
        x[2 * k + 1] = to_float<T>(v[k] >> 16);
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = c + k < cols ? to_float<T>(p[k]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(void* row, int64_t c, int64_t cols, bool wide,
                                       const float (&x)[8]) {
  if constexpr (std::is_same_v<T, F32>) {
    float* p = static_cast<float*>(row) + c;
    if (c + 8 <= cols) {  // any row is a multiple of 4 bytes
      *reinterpret_cast<f32x4_any*>(p) = f32x4_any{x[0], x[1], x[2], x[3]};
      *reinterpret_cast<f32x4_any*>(p + 4) = f32x4_any{x[4], x[5], x[6], x[7]};
      return;
    }
    for (int k = 0; k < 8; ++k)
      if (c + k < cols) p[k] = x[k];
  } else {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = from_float<T>(x[2 * k]) | (from_float<T>(x[2 * k + 1]) << 16);
    store_eight(static_cast<uint16_t*>(row) + c, v, cols - c, wide);
  }
}

// The place of a lane's eight values: part 0 .. 3 of group `at`, groups numbered through all
// rows, of which each has `groups`.  kFlat: rows follow each other without a gap and are whole
// groups, so the array is one row (a division less a group).
template <typename T, bool kFlat>
struct At {
  int64_t row, c;
  __device__ __forceinline__ At(int64_t at, int64_t groups, int part) {
    row = kFlat ? 0 : (uint64_t)at < (uint64_t(1) << 32) && groups < (int64_t(1) << 32)
                          ? (int64_t)((uint32_t)at / (uint32_t)groups)
                          : at / groups;
    c = (kFlat ? at : at - row * groups) * kGroup + 8 * part;
  }
};

// kPer groups per quad of lanes, kQuads apart: all loads of a lane before the first use.  Four
// where they still fill the chip (16384 x 3072 BF16, pack and unpack: 55 us with one, 51 with four), one for less work.
constexpr int kQuads = kThreads / 4;
constexpr int64_t kMany = 4 * 256 * 8 * kQuads;  // groups: eight workgroups of four per CU

template <typename T, bool kFlat, int kPer>
__global__ __launch_bounds__(kThreads) void act_pack_kernel(const void* __restrict__ src, int64_t cols,
                                                            int64_t ld, uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ exponents,
                                                            int64_t groups, int64_t total, bool wide) {
  const int part = threadIdx.x & 3;
  const int64_t first = (int64_t)blockIdx.x * kPer * kQuads + (threadIdx.x >> 2);
  float x[kPer][8];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t at = first + i * kQuads;
    const At<T, kFlat> p(at < total ? at : total - 1, groups, part);
    load8<T>(static_cast<const char*>(src) + p.row * ld * Fmt<T>::bytes, p.c, kFlat ? total * kGroup : cols, wide,
             x[i]);
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t at = first + i * kQuads;
    if (at >= total) return;  // whole quads leave together
    uint32_t w[2];
    const int e = act_encode<8>(x[i], w, [](uint32_t m) { return quad_max(m); });
    *reinterpret_cast<u32x2*>(codes + at * kGroup + 8 * part) = u32x2{w[0], w[1]};
    if (part == 0) exponents[at] = (uint8_t)e;
  }
}

template <typename T, bool kFlat, int kPer>
__global__ __launch_bounds__(kThreads) void act_unpack_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ exponents,
                                                              int64_t cols, void* __restrict__ dst,
                                                              int64_t ld, int64_t groups, int64_t total,
                                                              bool wide, bool saturate) {
  const int part = threadIdx.x & 3;
  const int64_t first = (int64_t)blockIdx.x * kPer * kQuads + (threadIdx.x >> 2);
  u32x2 w[kPer];
  uint32_t e[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t at = first + i * kQuads < total ? first + i * kQuads : total - 1;
    w[i] = *reinterpret_cast<const u32x2*>(codes + at * kGroup + 8 * part);
    e[i] = exponents[at];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t at = first + i * kQuads;
    if (at >= total) return;
    const At<T, kFlat> p(at, groups, part);
    const float scale = act_scale((int)e[i]);
    float lo[4], hi[4];
    act_decode4(w[i].x, scale, lo);
    act_decode4(w[i].y, scale, hi);
    float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    if (saturate && __any((int)e[i] >= kActTop<T>)) act_saturate<T>(x);
    store8<T>(static_cast<char*>(dst) + p.row * ld * Fmt<T>::bytes, p.c, kFlat ? total * kGroup : cols, wide, x);
  }
}

bool misaligned(const void* p, uintptr_t by) { return reinterpret_cast<uintptr_t>(p) % by != 0; }

// MORPH_OK with the number of groups and workgroups, or the status to return.
int act_shape(const void* values, int dtype, int64_t rows, int64_t cols, int64_t ld,
              const uint8_t* codes, const uint8_t* exponents, int64_t& groups, int64_t& total,
              int64_t& grid, int& per, bool& wide) {
  if (rows < 0 || cols < 0 || ld < cols) return MORPH_EINVAL;
  if (dtype != MORPH_DTYPE_F32 && dtype != MORPH_DTYPE_F16 && dtype != MORPH_DTYPE_BF16)
    return MORPH_EDTYPE;
  grid = 0;
  if (rows == 0 || cols == 0) return MORPH_OK;
  const int64_t size = dtype == MORPH_DTYPE_F32 ? 4 : 2;
  if (values == nullptr || codes == nullptr || exponents == nullptr || misaligned(codes, 8) ||
      misaligned(values, size))
    return MORPH_EINVAL;
  // the last element's byte offset and the grid
  if (ld > (INT64_MAX >> 4) / rows) return MORPH_ERANGE;
  groups = (cols + kGroup - 1) / kGroup;
  total = rows * groups;
  per = total >= kMany ? 4 : 1;
  grid = (total + per * kQuads - 1) / (per * kQuads);
  if (!launchable(grid, kThreads)) return MORPH_ERANGE;
  wide = !misaligned(values, 16) && (rows == 1 || ld * size % 16 == 0);
  return MORPH_OK;
}

// F(T, rows without gaps, groups per quad).
template <typename F>
void by_type(int dtype, bool flat, int per, F&& f) {
  auto with = [&](auto type) {
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 4> four;
    if (flat && per == 4) f(type, std::true_type{}, four);
    else if (flat) f(type, std::true_type{}, one);
    else if (per == 4) f(type, std::false_type{}, four);
    else f(type, std::false_type{}, one);
  };
  if (dtype == MORPH_DTYPE_F32) with(F32{});
  else if (dtype == MORPH_DTYPE_F16) with(F16{});
  else with(BF16{});
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" int morph_act_pack(const void* src, int dtype, int64_t rows, int64_t cols, int64_t ld,
                              uint8_t* codes, uint8_t* exponents, void* stream) {
  int64_t groups, total, grid;
  int per;
  bool wide;
  const int status = act_shape(src, dtype, rows, cols, ld, codes, exponents, groups, total, grid, per, wide);
  if (status != MORPH_OK || grid == 0) return status;
  by_type(dtype, ld == cols && cols % kGroup == 0, per, [&](auto type, auto flat, auto count) {
    hipLaunchKernelGGL((act_pack_kernel<decltype(type), decltype(flat)::value, decltype(count)::value>),
                       dim3((unsigned)grid), dim3(kThreads), 0, as_stream(stream), src, cols, ld, codes, exponents, groups, total, wide);
  });
  return launch_status();
}

extern "C" int morph_act_unpack(const uint8_t* codes, const uint8_t* exponents, int64_t rows,
                                int64_t cols, void* dst, int dtype, int64_t ld, void* stream) {
  int64_t groups, total, grid;
  int per;
  bool wide;
  const bool saturate = dtype >= 0 && (dtype & MORPH_ACT_SATURATE) != 0;
  if (saturate) dtype &= ~MORPH_ACT_SATURATE;
  const int status = act_shape(dst, dtype, rows, cols, ld, codes, exponents, groups, total, grid, per, wide);
  if (status != MORPH_OK || grid == 0) return status;
  by_type(dtype, ld == cols && cols % kGroup == 0, per, [&](auto type, auto flat, auto count) {
    hipLaunchKernelGGL((act_unpack_kernel<decltype(type), decltype(flat)::value, decltype(count)::value>),
                       dim3((unsigned)grid), dim3(kThreads), 0, as_stream(stream), codes, exponents, cols, dst, ld, groups, total, wide,
                       saturate);
  });
  return launch_status();
}
