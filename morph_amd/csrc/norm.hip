// Layer norm (morph_state_space.h) and its backward pass.
//
// A row is read once and stays in registers: a wave or a workgroup has it, 16 bytes a lane and access, finds the
// mean, then the variance around that mean, and writes y.  The backward reads x and dy, sums g and g xh over the row
// and writes dx; each workgroup takes many rows and keeps its lanes' columns of dweight and dbias in
// registers over all of them, then writes them as one row of partial sums, which a second launch adds up in
// a fixed order.  HBM bounds both.
#include "stage.h"

namespace morph {
namespace {

// Workgroups of a launch, each of which loads its next row before it sums the present one and its weights once.
// 16384 rows of 4096 in BF16, forward: 46.5 us with six on a CU (1024: 47.6, 2048: 49.7, one a row 60), backward 80.5
// with two (384: 85, 768: 83, 1024: 92; each leaves a row of partial sums).
constexpr int kForwardGroups = 1536;
constexpr int kBackGroups = 512;
constexpr int64_t kMostRowBlocks = int64_t(1) << 20;

// Sums of two values over the kThreads lanes that share a row (a wave, or the workgroup).
template <int kThreads>
struct RowSums {
  static constexpr int kW = kThreads / 64;
  float* slots;  // [2][kW][2] in LDS
  int turn = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    a = wave_sum(a), b = wave_sum(b);
    if constexpr (kW > 1) {
      float* s = slots + turn * kW * 2;
      const int w = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0) s[2 * w] = a, s[2 * w + 1] = b;
      __syncthreads();
      a = b = 0.0f;
#pragma unroll
      for (int i = 0; i < kW; ++i) a += s[2 * i], b += s[2 * i + 1];
      turn ^= 1;  // the other half is free: every wave has passed the barrier behind its last use
    }
  }
};

// kCount weights from c on; all: there are so many, else the first n, 0 behind them.
template <typename W, int kCount>
__device__ __forceinline__ void load_weights(const void* p, int64_t c, int64_t n, float none, float (&w)[kCount]) {
  constexpr int V = Wide<W>::kCount;
  static_assert(kCount % V == 0 || V % kCount == 0, "whole accesses, or a part of one");
  if (!p) {
#pragma unroll
    for (int k = 0; k < kCount; ++k) w[k] = none;
  } else if constexpr (V <= kCount) {
#pragma unroll
    for (int k = 0; k < kCount; k += V) {
      float x[V];
      Wide<W>::unpack(Wide<W>::load(p, c + k, n - k), x);
#pragma unroll
      for (int j = 0; j < V; ++j) w[k + j] = x[j];
    }
  } else {
#pragma unroll
    for (int k = 0; k < kCount; ++k) w[k] = k < n ? load_one<W>(p, c + k) : 0.0f;
  }
}

// Rows of at most kThreads * kIters * Wide<T>::kCount values, kWhole: a multiple of Wide<T>::kCount, so that a lane's
// values are all there or none of them is (the tests for each would take two instructions a value and the
// scalar registers for their results); a workgroup of 256 lanes has four rows at kThreads = 64.
template <typename T, typename W, int kThreads, int kIters, bool kWhole>
__global__ __launch_bounds__(kThreads == 64 ? 256 : kThreads) void norm_kernel(const morph_norm a, void* __restrict__ y,
                                                                              float* __restrict__ stats) {
  constexpr int V = Wide<T>::kCount, kRows = kThreads == 64 ? 4 : 1;
  __shared__ float slots[2 * (kThreads / 64) * 2];
  RowSums<kThreads> sums{slots};
  const int t = kThreads == 64 ? threadIdx.x & 63 : threadIdx.x;
  const float inverse = 1.0f / (float)a.cols;
  // In a workgroup of 1024 lanes the weights are read again for each row: see norm_back_kernel.
  constexpr bool kKeep = kThreads < 1024;
  float w[kKeep ? kIters : 1][V], b[kKeep ? kIters : 1][V];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int64_t c = (int64_t)(i * kThreads + t) * V;
      if (c >= a.cols) continue;
      load_weights<W, V>(a.weight, c, kWhole ? V : a.cols - c, 1.0f, w[i]);
      load_weights<W, V>(a.bias, c, kWhole ? V : a.cols - c, 0.0f, b[i]);
    }
  }
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + (kThreads == 64 ? threadIdx.x >> 6 : 0);
  u32x4 raw[kIters];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int64_t c = (int64_t)(i * kThreads + t) * V;
      raw[i] = 0;
      if (c < a.cols) raw[i] = Wide<T>::load(a.x, at * a.x_ld + c, kWhole ? V : a.cols - c);
    }
  };
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += step) {
    float x[kIters][V];
    float sum = 0.0f, none = 0.0f, squares = 0.0f;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      Wide<T>::unpack(raw[i], x[i]);
#pragma unroll
      for (int k = 0; k < V; ++k) sum += x[i][k];
    }
    if (row + step < a.rows) fetch(row + step);
    sums(sum, none);
    const float mean = sum * inverse;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int64_t c = (int64_t)(i * kThreads + t) * V;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        x[i][k] = c + (kWhole ? 0 : k) < a.cols ? x[i][k] - mean : 0.0f;
        squares = __fmaf_rn(x[i][k], x[i][k], squares);
      }
    }
    sums(squares, none);
    const float r = 1.0f / __builtin_sqrtf(squares * inverse + a.eps);
    if (stats && t == 0) stats[row] = mean, stats[a.rows + row] = r;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int64_t c = (int64_t)(i * kThreads + t) * V;
      if (c >= a.cols) continue;
      float wi[V], bi[V];
#pragma unroll
      for (int k = 0; k < V; ++k) wi[k] = w[kKeep ? i : 0][k], bi[k] = b[kKeep ? i : 0][k];
      if constexpr (!kKeep) {
        load_weights<W, V>(a.weight, c, kWhole ? V : a.cols - c, 1.0f, wi);
        load_weights<W, V>(a.bias, c, kWhole ? V : a.cols - c, 0.0f, bi);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) x[i][k] = __fmaf_rn(x[i][k] * r, wi[k], bi[k]);
      Wide<T>::store(y, row * a.cols + c, Wide<T>::pack(x[i]), kWhole ? V : a.cols - c);
    }
  }
}

// Rows of any length, read three times (from the caches, the last two).
template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_long_kernel(const morph_norm a, void* __restrict__ y,
                                                         float* __restrict__ stats) {
  __shared__ float slots[2 * 16 * 2];
  RowSums<1024> sums{slots};
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float sum = 0.0f, none = 0.0f, squares = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += 1024) sum += load_one<T>(a.x, row * a.x_ld + c);
    sums(sum, none);
    const float mean = sum / (float)a.cols;
    for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
      const float d = load_one<T>(a.x, row * a.x_ld + c) - mean;
      squares = __fmaf_rn(d, d, squares);
    }
    sums(squares, none);
    const float r = 1.0f / __builtin_sqrtf(squares / (float)a.cols + a.eps);
    if (stats && threadIdx.x == 0) stats[row] = mean, stats[a.rows + row] = r;
    for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
      const float w = a.weight ? load_one<W>(a.weight, c) : 1.0f, b = a.bias ? load_one<W>(a.bias, c) : 0.0f;
      store_one<T>(y, row * a.cols + c, __fmaf_rn((load_one<T>(a.x, row * a.x_ld + c) - mean) * r, w, b));
    }
  }
}

// parts: [gridDim.x][2][cols], this workgroup's rows of dweight and dbias.
template <typename T, typename W, int kThreads, int kIters, bool kWhole>
__global__ __launch_bounds__(kThreads == 64 ? 256 : kThreads) void norm_back_kernel(
    const morph_norm a, const float* __restrict__ stats, const void* __restrict__ dy, int64_t dy_ld,
    void* __restrict__ dx, float* __restrict__ parts) {
  constexpr int V = Wide<T>::kCount, kRows = kThreads == 64 ? 4 : 1;
  __shared__ float slots[2 * (kThreads / 64) * 2];
  RowSums<kThreads> sums{slots};
  const int t = kThreads == 64 ? threadIdx.x & 63 : threadIdx.x;
  const float inverse = 1.0f / (float)a.cols;
  // In a workgroup of 1024 lanes a lane has 128 registers: it reads the weights again for each row.
  constexpr bool kKeep = kThreads < 1024;
  float w[kKeep ? kIters : 1][V], dw[kIters][V], db[kIters][V];
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int64_t c = (int64_t)(i * kThreads + t) * V;
    if constexpr (kKeep) {
#pragma unroll
      for (int k = 0; k < V; ++k) w[i][k] = 0.0f;
      if (c < a.cols) load_weights<W, V>(a.weight, c, kWhole ? V : a.cols - c, 1.0f, w[i]);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.0f;
  }
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + (kThreads == 64 ? threadIdx.x >> 6 : 0);
  u32x4 rx[kIters], rd[kIters];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int64_t c = (int64_t)(i * kThreads + t) * V;
      rx[i] = rd[i] = 0;
      if (c < a.cols) {
        rx[i] = Wide<T>::load(a.x, at * a.x_ld + c, kWhole ? V : a.cols - c);
        rd[i] = Wide<T>::load(dy, at * dy_ld + c, kWhole ? V : a.cols - c);
      }
    }
  };
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += step) {
    const float mean = stats[row], r = stats[a.rows + row];
    float x[kIters][V], g[kIters][V];
    float sg = 0.0f, sx = 0.0f;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      Wide<T>::unpack(rx[i], x[i]);
      Wide<T>::unpack(rd[i], g[i]);
    }
    if (row + step < a.rows) fetch(row + step);
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      float fresh[V] = {};
      if constexpr (!kKeep) {
        const int64_t c = (int64_t)(i * kThreads + t) * V;
        if (c < a.cols) load_weights<W, V>(a.weight, c, kWhole ? V : a.cols - c, 1.0f, fresh);
      }
      const float(&wi)[V] = kKeep ? w[kKeep ? i : 0] : fresh;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        // dy and so g are 0 behind the row's end, and x is not looked at there
        x[i][k] = (x[i][k] - mean) * r;
        dw[i][k] = __fmaf_rn(g[i][k], x[i][k], dw[i][k]);
        db[i][k] += g[i][k];
        g[i][k] *= wi[k];
        sg += g[i][k];
        sx = __fmaf_rn(g[i][k], x[i][k], sx);
      }
    }
    sums(sg, sx);
    sg *= inverse, sx *= inverse;
#pragma unroll
    for (int i = 0; i < kIters; ++i) {
      const int64_t c = (int64_t)(i * kThreads + t) * V;
      if (c >= a.cols) continue;
#pragma unroll
      for (int k = 0; k < V; ++k) x[i][k] = r * (__fmaf_rn(-x[i][k], sx, g[i][k]) - sg);
      Wide<T>::store(dx, row * a.cols + c, Wide<T>::pack(x[i]), kWhole ? V : a.cols - c);
    }
  }
  if (!parts) return;
  float* mine = parts + (int64_t)blockIdx.x * 2 * a.cols;
  if constexpr (kThreads == 64) {  // the four waves' columns, joined in the waves' order
    __shared__ float join[2][64 * kIters * V];
    for (int wave = 0; wave < 4; ++wave) {
      if ((int)(threadIdx.x >> 6) == wave) {
#pragma unroll
        for (int i = 0; i < kIters; ++i)
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const int at = (i * V + k) * 64 + t;  // a bank a lane
            join[0][at] = dw[i][k] += wave ? join[0][at] : 0.0f;
            join[1][at] = db[i][k] += wave ? join[1][at] : 0.0f;
          }
      }
      __syncthreads();
    }
    if (threadIdx.x >> 6 != 3) return;
  }
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int64_t c = (int64_t)(i * kThreads + t) * V;
    if (c >= a.cols) continue;
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      Wide<F32>::store(mine, c + k, __builtin_bit_cast(u32x4, f32x4{dw[i][k], dw[i][k + 1], dw[i][k + 2], dw[i][k + 3]}),
                       a.cols - c - k);
      Wide<F32>::store(mine, a.cols + c + k,
                       __builtin_bit_cast(u32x4, f32x4{db[i][k], db[i][k + 1], db[i][k + 2], db[i][k + 3]}), a.cols - c - k);
    }
  }
}

// Rows of any length: the sums of dweight and dbias stay in this workgroup's row of parts.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void norm_long_back_kernel(const morph_norm a, const float* __restrict__ stats,
                                                              const void* __restrict__ dy, int64_t dy_ld,
                                                              void* __restrict__ dx, float* __restrict__ parts) {
  __shared__ float slots[2 * 16 * 2];
  RowSums<1024> sums{slots};
  float* mine = parts ? parts + (int64_t)blockIdx.x * 2 * a.cols : nullptr;
  bool fresh = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = stats[row], r = stats[a.rows + row];
    float sg = 0.0f, sx = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
      const float d = load_one<T>(dy, row * dy_ld + c), xh = (load_one<T>(a.x, row * a.x_ld + c) - mean) * r;
      const float g = d * (a.weight ? load_one<W>(a.weight, c) : 1.0f);
      sg += g;
      sx = __fmaf_rn(g, xh, sx);
      if (mine) {
        mine[c] = __fmaf_rn(d, xh, fresh ? 0.0f : mine[c]);
        mine[a.cols + c] = d + (fresh ? 0.0f : mine[a.cols + c]);
      }
    }
    fresh = false;
    sums(sg, sx);
    sg /= (float)a.cols, sx /= (float)a.cols;
    for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
      const float xh = (load_one<T>(a.x, row * a.x_ld + c) - mean) * r;
      const float g = load_one<T>(dy, row * dy_ld + c) * (a.weight ? load_one<W>(a.weight, c) : 1.0f);
      store_one<T>(dx, row * a.cols + c, r * (__fmaf_rn(-xh, sx, g) - sg));
    }
  }
}

// dweight and dbias: the sums of `count` rows of parts, 16 stretches of them side by side.
template <typename W>
__global__ __launch_bounds__(1024) void norm_sum_kernel(const float* __restrict__ parts, int count, int64_t cols,
                                                        void* __restrict__ dweight, void* __restrict__ dbias) {
  __shared__ float join[16][64];
  const int lane = threadIdx.x & 63, stretch = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  void* out = blockIdx.y ? dbias : dweight;
  if (!out) return;  // the whole workgroup
  float sum = 0.0f;
  if (c < cols) {
    const int each = (count + 15) / 16, from = stretch * each, to = from + each < count ? from + each : count;
    const float* p = parts + (int64_t)blockIdx.y * cols + c;
#pragma unroll 8
    for (int i = from; i < to; ++i) sum += p[(int64_t)i * 2 * cols];
  }
  join[stretch][lane] = sum;
  __syncthreads();
  if (stretch != 0 || c >= cols) return;
  sum = join[0][lane];
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += join[i][lane];
  store_one<W>(out, c, sum);
}

// Lanes for a row, accesses of each and whether the last is whole: f of the first that holds it, else of
// (0, 1, false).
template <typename F>
int by_length(int64_t cols, int wide, F&& g) {
  const int64_t n = (cols + wide - 1) / wide;  // accesses of a row
  auto f = [&](auto threads, auto iters) {
    return cols % wide ? g(threads, iters, std::false_type{}) : g(threads, iters, std::true_type{});
  };
  typedef std::integral_constant<int, 64> Wave;
  typedef std::integral_constant<int, 256> Group;
  typedef std::integral_constant<int, 1024> Large;
  typedef std::integral_constant<int, 1> One;
  typedef std::integral_constant<int, 2> Two;
  typedef std::integral_constant<int, 4> Four;
  if (n <= 64) return f(Wave{}, One{});
  if (n <= 128) return f(Wave{}, Two{});
  if (n <= 256) return f(Group{}, One{});
  if (n <= 512) return f(Group{}, Two{});
  if (n <= 1024) return f(Group{}, Four{});
  if (n <= 2048) return f(Large{}, Two{});
  return g(std::integral_constant<int, 0>{}, One{}, std::false_type{});
}

int64_t back_groups(int64_t rows) { return rows < kBackGroups ? (rows > 0 ? rows : 1) : kBackGroups; }

int check(const morph_norm* a, int dtype) {
  if (!a || a->rows < 0 || a->cols < 0 || !(a->eps >= 0)) return MORPH_EINVAL;
  if (!known_dtype(dtype) || (a->weight_dtype != MORPH_DTYPE_F32 && a->weight_dtype != dtype)) return MORPH_EDTYPE;
  if (a->rows > 0 && a->cols > 0 && (!a->x || a->x_ld < (a->rows > 1 ? a->cols : 0))) return MORPH_EINVAL;
  return MORPH_OK;
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" int morph_norm_forward(const morph_norm* a, int dtype, void* y, float* stats, void* stream) {
  if (const int rc = check(a, dtype)) return rc;
  if (a->rows == 0 || a->cols == 0) return MORPH_OK;
  if (!y) return MORPH_EINVAL;
  hipStream_t s = as_stream(stream);
  return by_dtypes(dtype, a->weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    return by_length(a->cols, Wide<T>::kCount, [&](auto threads, auto iters, auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      constexpr int kThreads = decltype(threads)::value, kIters = decltype(iters)::value;
      if constexpr (kThreads == 0) {
        const int64_t blocks = a->rows < kMostRowBlocks ? a->rows : kMostRowBlocks;
        hipLaunchKernelGGL((norm_long_kernel<T, W>), dim3((unsigned)blocks), dim3(1024), 0, s, *a, y, stats);
      } else {
        constexpr int kRows = kThreads == 64 ? 4 : 1;
        int64_t blocks = (a->rows + kRows - 1) / kRows;
        if (blocks > kForwardGroups) blocks = kForwardGroups;
        hipLaunchKernelGGL((norm_kernel<T, W, kThreads, kIters, kWhole>), dim3((unsigned)blocks),
                           dim3(kThreads == 64 ? 256 : kThreads), 0, s, *a, y, stats);
      }
      return launch_status();
    });
  });
}

extern "C" size_t morph_norm_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 0) return 0;
  return (size_t)back_groups(rows) * 2 * (size_t)cols * sizeof(float);
}

extern "C" int morph_norm_backward(const morph_norm* a, int dtype, const float* stats, const void* dy, int64_t dy_ld,
                                   void* dx, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  if (const int rc = check(a, dtype)) return rc;
  if (a->cols == 0) return MORPH_OK;
  if (a->rows > 0 && (!stats || !dy || !dx || dy_ld < (a->rows > 1 ? a->cols : 0))) return MORPH_EINVAL;
  const bool sums = dweight || dbias;
  if (sums && (!workspace || workspace_bytes < morph_norm_workspace_bytes(a->rows, a->cols))) return MORPH_EWORKSPACE;
  const int64_t sum_blocks = (a->cols + 63) / 64;
  if (!launchable(sum_blocks, 1024)) return MORPH_ERANGE;
  float* parts = sums ? static_cast<float*>(workspace) : nullptr;
  hipStream_t s = as_stream(stream);
  return by_dtypes(dtype, a->weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    int groups = 0;
    int rc = a->rows == 0 ? MORPH_OK : by_length(a->cols, Wide<T>::kCount, [&](auto threads, auto iters, auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      constexpr int kThreads = decltype(threads)::value, kIters = decltype(iters)::value;
      if constexpr (kThreads == 0) {
        groups = (int)back_groups(a->rows);
        hipLaunchKernelGGL((norm_long_back_kernel<T, W>), dim3(groups), dim3(1024), 0, s, *a, stats, dy, dy_ld, dx, parts);
      } else {
        constexpr int kRows = kThreads == 64 ? 4 : 1;
        groups = (int)back_groups((a->rows + kRows - 1) / kRows);
        hipLaunchKernelGGL((norm_back_kernel<T, W, kThreads, kIters, kWhole>), dim3(groups), dim3(kThreads == 64 ? 256 : kThreads),
                           0, s, *a, stats, dy, dy_ld, dx, parts);
      }
      return launch_status();
    });
    if (rc != MORPH_OK || !sums) return rc;
    hipLaunchKernelGGL(norm_sum_kernel<W>, dim3((unsigned)sum_blocks, 2), dim3(1024), 0, s, parts, groups, a->cols, dweight,
                       dbias);
    return launch_status();
  });
}
