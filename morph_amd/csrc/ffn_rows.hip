// The gated feed-forward block's products for few rows (a token, or a batch of them being
// written): the weights cross once and bound the time, 113 MB for d = 3072, ff = 6144.
//
// A workgroup takes some rows of the weights and all of K; its waves take blocks of 64 k in turn,
// so that a wave's two loads per weight row cover whole 128-byte lines and the workgroup walks
// along its rows.  Fragments go from memory straight to v_mfma_f32_16x16x32 with the weights as
// the first operand and up to 16 rows of P as the second (more in further accumulators): no
// weight passes through LDS.  The waves' sums meet in LDS, in wave order.
//
// Up to 16 rows of P the gate's workgroup holds 8 rows of each matrix, the halves of one fragment
// (768 workgroups for ff = 6144, all resident); else a workgroup holds 16 rows.  Measured, us,
// for d = 3072, ff = 6144: gate with 8 / 16 rows 14.7 / 17.4 for one row of P, 21.9 / 21.1 for
// 16, 29.1 / 26.7 for 32; down with the same 8 rows twice 15.9, 16 rows 9.5.  4, 8 or 16 waves
// and 3 or 6 blocks in flight: within 5%, 16 waves up to 40% slower.  75 and 38 MB in 14.7 and
// 9.5 us are 5.1 and 4.0 TB/s with each launch's fill and drain.
//
// Loads need no alignment beyond the elements' own, so odd widths and views run the same code; the
// block of K that is not whole is loaded value by value.  Rows at odd elements (kOdd) are loaded
// from the 4-byte boundary before and shifted: 16-byte loads take any address, but at
// 2 mod 4 take about five times as long (50 rows of 1857 x 5198 64 us against 33-37).
#include "ffn_rows.h"

namespace morph {
namespace {

typedef uint32_t u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));

// Eight values at p as loaded.  kOdd: the four words from the boundary at or before p (a value
// more in front, of the row before or the same allocation), and behind them the last value.
template <bool kOdd>
struct Eight {
  u32x4 w;
  __device__ __forceinline__ void load(const uint16_t* p) { w = *reinterpret_cast<const u32x4_any2*>(p); }
  __device__ __forceinline__ u32x4 values(uint32_t) const { return w; }
};
template <>
struct Eight<true> {
  u32x4 w;
  uint32_t last;
  __device__ __forceinline__ void load(const uint16_t* p) {
    w = *reinterpret_cast<const u32x4_any2*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
    last = p[7];
  }
  __device__ __forceinline__ u32x4 values(uint32_t shift) const {  // 16 for an odd row, else 0
    return u32x4{__builtin_amdgcn_alignbit(w.y, w.x, shift), __builtin_amdgcn_alignbit(w.z, w.y, shift),
                 __builtin_amdgcn_alignbit(w.w, w.z, shift), __builtin_amdgcn_alignbit(last, w.w, shift)};
  }
};
// Values k .. k + 7 of a row of K.
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
// kRows: weight rows of a workgroup, of each matrix: 8 (kGated: the halves of one fragment) or 16.
template <typename T, bool kGated, int kTiles, int kWaves, int kBlocks, int kRows, bool kOdd>
__global__ __launch_bounds__(64 * kWaves) void ffn_few_rows_kernel(
    const uint16_t* __restrict__ P, int64_t ldp, const uint16_t* __restrict__ Q0, int64_t ldq0,
    const uint16_t* __restrict__ Q1, int64_t ldq1, int64_t M, int64_t N, int64_t K, uint16_t* __restrict__ C,
    int64_t ldc) {
  constexpr bool kHalves = kRows == 8;
  constexpr int kQ = kGated && !kHalves ? 2 : 1;
  __shared__ f32x4 sums[kWaves][kQ][kTiles][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * kRows;
  const int64_t qat = n0 + (lane & (kRows - 1)), qrow = qat < N ? qat : N - 1;  // rows past the end are not stored
  const int k0 = 8 * (lane >> 4);
  const uint16_t* q[kQ];
  static_assert(kGated || !kHalves, "the halves are gate and up");
  if constexpr (kHalves) {
    q[0] = (lane & 8) ? Q1 + qrow * ldq1 : Q0 + qrow * ldq0;
  } else {
    q[0] = Q0 + qrow * ldq0;
    if constexpr (kGated) q[1] = Q1 + qrow * ldq1;
  }
  const uint16_t* p[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int64_t row = 16 * t + (lane & 15);
    p[t] = P + (row < M ? row : M - 1) * ldp;
  }
  f32x4 acc[kQ][kTiles] = {};
  auto shift = [](const uint16_t* row) { return (uint32_t)(reinterpret_cast<uintptr_t>(row) & 2) * 8; };
  // `blocks` blocks of 64 k from block `at` on, every load before the first wait
  auto run = [&](int64_t at, auto blocks) {
    constexpr int kCount = decltype(blocks)::value;
    Eight<kOdd> a[kCount][2][kQ], b[kCount][2][kTiles];
#pragma unroll
    for (int u = 0; u < kCount; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t k = (at + u * kWaves) * 64 + 32 * h + k0;
#pragma unroll
        for (int i = 0; i < kQ; ++i) a[u][h][i].load(q[i] + k);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) b[u][h][t].load(p[t] + k);
      }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kCount; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < kQ; ++i)
#pragma unroll
          for (int t = 0; t < kTiles; ++t)
            acc[i][t] = mfma16<T>(a[u][h][i].values(shift(q[i])), b[u][h][t].values(shift(p[t])), acc[i][t]);
  };
  const int64_t whole = K / 64;
  int64_t at = wave;
  for (; at + (kBlocks - 1) * kWaves < whole; at += kBlocks * kWaves)
    run(at, std::integral_constant<int, kBlocks>{});
  for (; at < whole; at += kWaves) run(at, std::integral_constant<int, 1>{});
  if (at == whole && K % 64 != 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t k = whole * 64 + 32 * h + k0;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const u32x4 b = load_part(p[t], k, K);
#pragma unroll
        for (int i = 0; i < kQ; ++i) acc[i][t] = mfma16<T>(load_part(q[i], k, K), b, acc[i][t]);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < kQ; ++i)
#pragma unroll
    for (int t = 0; t < kTiles; ++t) sums[wave][i][t][lane] = acc[i][t];
  __syncthreads();
  if (wave >= kTiles) return;
  // wave t: rows 16 t + lane % 16 of P, columns n0 + 4 (lane / 16) .. + 3 (kHalves: of the first
  // 32 lanes; the second half of the fragment's rows is 32 lanes on)
  constexpr int kSums = kGated ? 2 : 1;
  f32x4 x[kSums];
#pragma unroll
  for (int i = 0; i < kSums; ++i) {
    const int from = kHalves ? (lane & 31) + 32 * i : lane, which = kHalves ? 0 : i;
    x[i] = sums[0][which][wave][from];
    for (int w = 1; w < kWaves; ++w) {
      const f32x4 y = sums[w][which][wave][from];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[i][r] += y[r];
    }
  }
  const int64_t row = 16 * wave + (lane & 15), col = n0 + 4 * (lane >> 4);
  if (row >= M || (kHalves && lane >= 32)) return;
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
  constexpr int kRows = kGated && kTiles == 1 ? 8 : 16;
  constexpr int kWaves = 4, kBlocks = kTiles == 1 ? 6 : kTiles == 2 ? 3 : 2;
  auto odd = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 4 != 0 || ld % 2 != 0; };
  const dim3 grid((unsigned)((N + kRows - 1) / kRows)), block(64 * kWaves);
  if (odd(Q0, ldq0) || (kGated && odd(Q1, ldq1)) || odd(P, M > 1 ? ldp : 0))
    hipLaunchKernelGGL((ffn_few_rows_kernel<T, kGated, kTiles, kWaves, kBlocks, kRows, true>), grid, block, 0, s,
                       P, ldp, Q0, ldq0, Q1, ldq1, M, N, K, C, ldc);
  else
    hipLaunchKernelGGL((ffn_few_rows_kernel<T, kGated, kTiles, kWaves, kBlocks, kRows, false>), grid, block, 0, s,
                       P, ldp, Q0, ldq0, Q1, ldq1, M, N, K, C, ldc);
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
