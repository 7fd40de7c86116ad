// The gated feed-forward block's products for few rows (a token, or a batch of them being
// written): the weights cross once and bound the time, 113 MB for d = 3072, ff = 6144.
//
// A workgroup takes 16 rows of the weights (of gate and up both) and all of K; its waves take
// blocks of 64 k in turn, so that a wave's two loads per weight row cover whole 128-byte lines
// and the workgroup walks along its rows.  Fragments go from memory straight to v_mfma_f32_16x16x32
// with the weights as the first operand and up to 16 rows of P as the second (more in further
// accumulators): no weight passes through LDS.  The waves' sums meet in LDS, in wave order.
//
// Loads need no alignment beyond the elements' own (global loads of 16 bytes take any
// address), so odd widths and views run the same code; the block of K that is not whole is
// loaded value by value.
#include "ffn_rows.h"

namespace morph {
namespace {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// Values k .. k + 7 of a row of K.
__device__ __forceinline__ u32x4 load_whole(const uint16_t* p) { return *reinterpret_cast<const u32x4_any*>(p); }
__device__ __forceinline__ u32x4 load_part(const uint16_t* row, int64_t k, int64_t K) {
  u32x4 v{0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < K) v[i >> 1] |= (uint32_t)row[k + i] << (16 * (i & 1));
  return v;
}

template <typename T>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same_v<T, F16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                   0, 0, 0);
}

// kTiles: 16-row tiles of P.  kBlocks: blocks of 64 k whose loads a wave has in flight.
template <typename T, bool kGated, int kTiles, int kWaves, int kBlocks>
__global__ __launch_bounds__(64 * kWaves) void ffn_few_rows_kernel(
    const uint16_t* __restrict__ P, int64_t ldp, const uint16_t* __restrict__ Q0, int64_t ldq0,
    const uint16_t* __restrict__ Q1, int64_t ldq1, int64_t M, int64_t N, int64_t K, uint16_t* __restrict__ C,
    int64_t ldc) {
  constexpr int kQ = kGated ? 2 : 1;
  __shared__ f32x4 sums[kWaves][kQ][kTiles][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t qrow = n0 + (lane & 15) < N ? n0 + (lane & 15) : N - 1;  // rows past the end are not stored
  const int k0 = 8 * (lane >> 4);
  const uint16_t* q[kQ];
  q[0] = Q0 + qrow * ldq0;
  if constexpr (kGated) q[1] = Q1 + qrow * ldq1;
  const uint16_t* p[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int64_t row = 16 * t + (lane & 15);
    p[t] = P + (row < M ? row : M - 1) * ldp;
  }
  f32x4 acc[kQ][kTiles] = {};
  auto block = [&](int64_t k, auto load) {
    u32x4 b[2][kTiles], a[2][kQ];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < kQ; ++i) a[h][i] = load(q[i], k + 32 * h + k0);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) b[h][t] = load(p[t], k + 32 * h + k0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kQ; ++i)
#pragma unroll
        for (int t = 0; t < kTiles; ++t) acc[i][t] = mfma16<T>(a[h][i], b[h][t], acc[i][t]);
  };
  const int64_t whole = K / 64;
  int64_t at = wave;
  for (; at + (kBlocks - 1) * kWaves < whole; at += kBlocks * kWaves) {
    u32x4 a[kBlocks][2][kQ], b[kBlocks][2][kTiles];
#pragma unroll
    for (int u = 0; u < kBlocks; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t k = (at + u * kWaves) * 64 + 32 * h + k0;
#pragma unroll
        for (int i = 0; i < kQ; ++i) a[u][h][i] = load_whole(q[i] + k);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) b[u][h][t] = load_whole(p[t] + k);
      }
    __builtin_amdgcn_sched_barrier(0);  // every load before the first wait
#pragma unroll
    for (int u = 0; u < kBlocks; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < kQ; ++i)
#pragma unroll
          for (int t = 0; t < kTiles; ++t) acc[i][t] = mfma16<T>(a[u][h][i], b[u][h][t], acc[i][t]);
  }
  for (; at < whole; at += kWaves) block(at * 64, [](const uint16_t* row, int64_t k) { return load_whole(row + k); });
  if (at == whole && K % 64 != 0)
    block(whole * 64, [&](const uint16_t* row, int64_t k) { return load_part(row, k, K); });

#pragma unroll
  for (int i = 0; i < kQ; ++i)
#pragma unroll
    for (int t = 0; t < kTiles; ++t) sums[wave][i][t][lane] = acc[i][t];
  __syncthreads();
  if (wave >= kTiles) return;
  // wave t: rows 16 t + lane % 16 of P, columns n0 + 4 (lane / 16) .. + 3
  f32x4 x[kQ];
#pragma unroll
  for (int i = 0; i < kQ; ++i) {
    x[i] = sums[0][i][wave][lane];
    for (int w = 1; w < kWaves; ++w) {
      const f32x4 y = sums[w][i][wave][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[i][r] += y[r];
    }
  }
  const int64_t row = 16 * wave + (lane & 15), col = n0 + 4 * (lane >> 4);
  if (row >= M) return;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float v = x[0][r];
    if constexpr (kGated) v = ffn_gate(v, x[1][r]);
    if (col + r < N) C[row * ldc + col + r] = (uint16_t)from_float<T>(v);
  }
}

template <typename T, bool kGated, int kTiles>
void launch_few(const uint16_t* P, int64_t ldp, const uint16_t* Q0, int64_t ldq0, const uint16_t* Q1, int64_t ldq1,
                int64_t M, int64_t N, int64_t K, uint16_t* C, int64_t ldc, hipStream_t s) {
  constexpr int kWaves = kGated ? 8 : 16, kBlocks = kTiles <= 2 ? 6 / kTiles : 2;
  hipLaunchKernelGGL((ffn_few_rows_kernel<T, kGated, kTiles, kWaves, kBlocks>), dim3((unsigned)((N + 15) / 16)),
                     dim3(64 * kWaves), 0, s, P, ldp, Q0, ldq0, Q1, ldq1, M, N, K, C, ldc);
}

template <typename T, bool kGated, typename... Args>
void launch_tiles_of(int64_t M, Args... args) {
  if (M <= 16) launch_few<T, kGated, 1>(args...);
  else if (M <= 32) launch_few<T, kGated, 2>(args...);
  else launch_few<T, kGated, 4>(args...);
}

}  // namespace
}  // namespace morph

int morph::ffn_few_rows(int dtype, bool gated, const uint16_t* P, int64_t ldp, const uint16_t* Q0, int64_t ldq0,
                        const uint16_t* Q1, int64_t ldq1, int64_t M, int64_t N, int64_t K, uint16_t* C, int64_t ldc,
                        hipStream_t s) {
  if (dtype == MORPH_DTYPE_F16) {
    if (gated) launch_tiles_of<F16, true>(M, P, ldp, Q0, ldq0, Q1, ldq1, M, N, K, C, ldc, s);
    else launch_tiles_of<F16, false>(M, P, ldp, Q0, ldq0, Q1, ldq1, M, N, K, C, ldc, s);
  } else {
    if (gated) launch_tiles_of<BF16, true>(M, P, ldp, Q0, ldq0, Q1, ldq1, M, N, K, C, ldc, s);
    else launch_tiles_of<BF16, false>(M, P, ldp, Q0, ldq0, Q1, ldq1, M, N, K, C, ldc, s);
  }
  return launch_status();
}
