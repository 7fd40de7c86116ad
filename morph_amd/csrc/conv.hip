// Short causal convolution along the steps with silu (morph_state_space.h), and its backward pass.
//
// A lane has a few neighbouring channels and walks a run of steps, the last taps - 1 inputs in registers: a row of x
// is read once by its run and once more by the next one's start.  The backward walks the same way taps - 1 steps
// further: p and so dp of a step come from the window of x again, the gradient of x from a window of dp, and the
// weights' gradients stay in registers over the run.  Workgroups take runs of several sequences so that at most
// kParts rows of partial sums are left for a second launch.  HBM bounds the forward; the backward takes some 30
// instructions an element, which cost as much as its bytes.
//
// kWhole: the channels come out in whole lanes, so that an access needs no test of its own.
#include "stage.h"

namespace morph {
namespace {

// 4 x 2048 steps of 5120 channels in BF16 with 4 taps: forward 36 us; backward 57.5 us (runs of 20 steps: 63, of 32: 62, of
// 40: 64; 8 steps ahead: 75; with 2 channels a lane: 68).
constexpr int kRun = 16;      // steps of a wave, forward
constexpr int kBackRun = 24;  // and backward
constexpr int kAhead = 4;     // steps whose loads are issued together, backward
constexpr int kParts = 512;   // rows of partial sums
constexpr int V = 4;          // channels of a lane

// V neighbouring channels at any element's address, as loaded (16 bits: two a word).
template <typename T>
struct Few {
  static constexpr int kWords = V * Fmt<T>::bytes / 4;
  typedef uint32_t raw __attribute__((ext_vector_type(kWords)));
  typedef uint32_t at_any __attribute__((ext_vector_type(kWords), aligned(Fmt<T>::bytes)));
  // The lane's part of the wave's channels, the first of which lies at `at`: a wave-uniform address, and an offset that the
  // access adds.
  static __device__ __forceinline__ const char* place(const void* p, int64_t at) {
    return static_cast<const char*>(p) + at * Fmt<T>::bytes + (threadIdx.x & 63) * (uint32_t)(V * Fmt<T>::bytes);
  }
  // The first n of them, the others 0.
  static __device__ __forceinline__ raw load(const void* p, int64_t at, int64_t n) {
    const char* q = place(p, at);
    if (n >= V) return *reinterpret_cast<const at_any*>(q);
    raw w = 0;
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) {
        if constexpr (Fmt<T>::bytes == 4) w[k] = reinterpret_cast<const uint32_t*>(q)[k];
        else w[k / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(q)[k] << (16 * (k % 2));
      }
    return w;
  }
  static __device__ __forceinline__ float value(const raw& w, int k) {
    if constexpr (Fmt<T>::bytes == 4) return __builtin_bit_cast(float, (uint32_t)w[k]);
    else return to_float<T>(k % 2 ? w[k / 2] >> 16 : w[k / 2] & 0xFFFFu);
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, int64_t n, const raw& w) {
    char* q = const_cast<char*>(place(p, at));
    if (n >= V) {
      *reinterpret_cast<at_any*>(q) = w;
      return;
    }
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < n) {
        if constexpr (Fmt<T>::bytes == 4) reinterpret_cast<uint32_t*>(q)[k] = w[k];
        else reinterpret_cast<uint16_t*>(q)[k] = (uint16_t)(w[k / 2] >> (16 * (k % 2)));
      }
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, int64_t n, const float (&x)[V]) {
    raw w;
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      if constexpr (Fmt<T>::bytes == 4) w[k] = __builtin_bit_cast(uint32_t, x[k]);
      else w[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
    }
    store(p, at, n, w);
  }
};

template <typename W, int kTaps>
__device__ __forceinline__ void load_taps(const morph_conv& a, int64_t c, int64_t n, float (&w)[kTaps][V],
                                          float (&bias)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = a.bias && i < n ? load_one<W>(a.bias, c + i) : 0.0f;
#pragma unroll
    for (int k = 0; k < kTaps; ++k) w[k][i] = i < n ? load_one<W>(a.weight, (c + i) * kTaps + k) : 0.0f;
  }
}

// x of step t of sequence b, where t may lie before the first step; 0 behind the last one.
template <typename T>
__device__ __forceinline__ typename Few<T>::raw load_input(const morph_conv& a, int64_t b, int64_t t, int64_t c,
                                                                int64_t n) {
  if (t >= 0) return t < a.steps ? Few<T>::load(a.x, b * a.x_batch + t * a.x_step + c, n) : typename Few<T>::raw(0);
  return a.before ? Few<T>::load(a.before, (b * (a.taps - 1) + t + a.taps - 1) * a.dim + c, n) : typename Few<T>::raw(0);
}

struct ConvGrid {
  int64_t channel_blocks, time_blocks;
};

template <typename T, typename W, int kTaps, bool kWhole>
__global__ __launch_bounds__(256) void conv_kernel(const morph_conv a, const ConvGrid g, void* __restrict__ y,
                                                   void* __restrict__ after) {
  const int64_t block = blockIdx.x, cb = block % g.channel_blocks, rest = block / g.channel_blocks;
  const int64_t tb = rest % g.time_blocks, b = rest / g.time_blocks;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t c = cb * 64 * V, mine = c + (threadIdx.x & 63) * V, n = kWhole ? V : a.dim - mine;
  if (mine >= a.dim) return;
  const int64_t t0 = (tb * 4 + wave) * kRun;
  typedef typename Few<T>::raw raw;
  if (t0 < a.steps) {
    raw x[kTaps - 1 + kRun];  // all of the run's loads first
    float w[kTaps][V], bias[V], in[kTaps][V];
    if (t0 + kRun <= a.steps) {
      const int64_t at = b * a.x_batch + t0 * a.x_step + c;
#pragma unroll
      for (int i = 0; i < kRun; ++i) x[kTaps - 1 + i] = Few<T>::load(a.x, at + i * a.x_step, n);
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i) x[kTaps - 1 + i] = load_input<T>(a, b, t0 + i, c, n);
    }
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k) x[k] = load_input<T>(a, b, t0 - (kTaps - 1) + k, c, n);
    load_taps<W, kTaps>(a, mine, n, w, bias);
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) in[k + 1][j] = Few<T>::value(x[k], j);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      if (t0 + i >= a.steps) break;
      float out[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int k = 0; k < kTaps - 1; ++k) in[k][j] = in[k + 1][j];
        in[kTaps - 1][j] = Few<T>::value(x[kTaps - 1 + i], j);
        float p = bias[j];
#pragma unroll
        for (int k = 0; k < kTaps; ++k) p = __fmaf_rn(w[k][j], in[k][j], p);
        out[j] = p * gate_sigmoid(p);
      }
      Few<T>::store(y, (b * a.steps + t0 + i) * a.dim + c, n, out);
    }
  }
  if (tb == g.time_blocks - 1 && wave == 0) {
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k)
      Few<T>::store(after, (b * (kTaps - 1) + k) * a.dim + c, n, load_input<T>(a, b, a.steps - (kTaps - 1) + k, c, n));
  }
}

// parts: [gridDim.y][taps + 1][dim].
template <typename T, typename W, int kTaps, bool kWhole>
__global__ __launch_bounds__(256) void conv_back_kernel(const morph_conv a, const ConvGrid g, const void* __restrict__ dy,
                                                        int64_t dy_batch, int64_t dy_step,
                                                        const void* __restrict__ dafter, void* __restrict__ dx,
                                                        void* __restrict__ dbefore, float* __restrict__ parts) {
  typedef typename Few<T>::raw raw;
  __shared__ float join[kTaps + 1][V][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.x * 64 * V, mine = c + lane * V, n = kWhole ? V : a.dim - mine;
  float w[kTaps][V], bias[V], dw[kTaps + 1][V];
  load_taps<W, kTaps>(a, mine, mine < a.dim ? n : 0, w, bias);
#pragma unroll
  for (int k = 0; k <= kTaps; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[k][j] = 0.0f;
  for (int64_t unit = blockIdx.y; unit < a.batch * g.time_blocks; unit += gridDim.y) {
    const int64_t b = unit / g.time_blocks, t0 = ((unit % g.time_blocks) * 4 + wave) * kBackRun;
    if (mine >= a.dim || (t0 >= a.steps && t0 > 0)) continue;
    const int64_t end = t0 + kBackRun + kTaps - 1;
    raw nx[kAhead], ny[kAhead];  // x and dy of the next steps
    auto fetch = [&](int64_t t) {
      if (t + kAhead <= a.steps && t + kAhead <= end) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          nx[i] = Few<T>::load(a.x, b * a.x_batch + (t + i) * a.x_step + c, n);
          ny[i] = Few<T>::load(dy, b * dy_batch + (t + i) * dy_step + c, n);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          nx[i] = load_input<T>(a, b, t + i, c, n);
          ny[i] = t + i < a.steps && t + i < end ? Few<T>::load(dy, b * dy_batch + (t + i) * dy_step + c, n) : raw(0);
        }
      }
    };
    float x[kTaps][V], d[kTaps][V];  // of the last kTaps steps; d is dp
    fetch(t0);
#pragma unroll
    for (int k = 0; k < kTaps - 1; ++k) {
      const raw in = load_input<T>(a, b, t0 - (kTaps - 1) + k, c, n);
#pragma unroll
      for (int j = 0; j < V; ++j) x[k + 1][j] = Few<T>::value(in, j), d[k + 1][j] = 0.0f;
    }
    for (int64_t t = t0; t < end && t < a.steps + kTaps - 1; t += kAhead) {
      raw rx[kAhead], ry[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) rx[i] = nx[i], ry[i] = ny[i];
      if (t + kAhead < end && t + kAhead < a.steps + kTaps - 1) fetch(t + kAhead);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const bool inside = t + i < t0 + kBackRun;
#pragma unroll
        for (int j = 0; j < V; ++j) {
#pragma unroll
          for (int k = 0; k < kTaps - 1; ++k) x[k][j] = x[k + 1][j], d[k][j] = d[k + 1][j];
          x[kTaps - 1][j] = Few<T>::value(rx[i], j);
          float p = bias[j];
#pragma unroll
          for (int k = 0; k < kTaps; ++k) p = __fmaf_rn(w[k][j], x[k][j], p);
          const float e = Few<T>::value(ry[i], j) * silu(p).slope;
          d[kTaps - 1][j] = e;
          if (inside) {
#pragma unroll
            for (int k = 0; k < kTaps; ++k) dw[k][j] = __fmaf_rn(e, x[k][j], dw[k][j]);
            dw[kTaps][j] += e;
          }
        }
        // the step whose last share this was
        const int64_t at = t + i - (kTaps - 1);
        if (at >= a.steps || at >= t0 + kBackRun || (at < t0 && t0 > 0)) continue;
        float out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          out[j] = 0.0f;
#pragma unroll
          for (int k = 0; k < kTaps; ++k) out[j] = __fmaf_rn(w[k][j], d[kTaps - 1 - k][j], out[j]);
        }
        if (dafter && at + kTaps - 1 >= a.steps) {
          const raw more = Few<T>::load(dafter, (b * (kTaps - 1) + at + kTaps - 1 - a.steps) * a.dim + c, n);
#pragma unroll
          for (int j = 0; j < V; ++j) out[j] += Few<T>::value(more, j);
        }
        if (at >= 0) Few<T>::store(dx, (b * a.steps + at) * a.dim + c, n, out);
        else if (dbefore) Few<T>::store(dbefore, (b * (kTaps - 1) + at + kTaps - 1) * a.dim + c, n, out);
      }
    }
  }
  for (int i = 0; i < 4; ++i) {  // in the waves' order
    if (wave == i) {
#pragma unroll
      for (int k = 0; k <= kTaps; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) join[k][j][lane] = dw[k][j] += i ? join[k][j][lane] : 0.0f;
    }
    __syncthreads();
  }
  if (wave != 3 || mine >= a.dim) return;
#pragma unroll
  for (int k = 0; k <= kTaps; ++k)
    Few<F32>::store(parts, ((int64_t)blockIdx.y * (kTaps + 1) + k) * a.dim + c, n, dw[k]);
}

template <typename W>
__global__ __launch_bounds__(1024) void conv_sum_kernel(const float* __restrict__ parts, int count, int64_t dim, int taps,
                                                        void* __restrict__ dweight, void* __restrict__ dbias) {
  __shared__ float join[16][64];
  const int lane = threadIdx.x & 63, stretch = threadIdx.x >> 6, k = blockIdx.y;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  void* out = k < taps ? dweight : dbias;
  if (!out) return;
  float sum = 0.0f;
  if (c < dim) {
    const int each = (count + 15) / 16, from = stretch * each, to = from + each < count ? from + each : count;
    const float* p = parts + (int64_t)k * dim + c;
#pragma unroll 8
    for (int i = from; i < to; ++i) sum += p[(int64_t)i * (taps + 1) * dim];
  }
  join[stretch][lane] = sum;
  __syncthreads();
  if (stretch != 0 || c >= dim) return;
  sum = join[0][lane];
#pragma unroll
  for (int i = 1; i < 16; ++i) sum += join[i][lane];
  store_one<W>(out, k < taps ? c * taps + k : c, sum);
}

// f(taps, whole) for whether lanes have all of their channels or none.
template <typename F>
int by_form(int taps, int64_t dim, F&& f) {
  auto whole = [&](auto k) { return dim % V ? f(k, std::false_type{}) : f(k, std::true_type{}); };
  switch (taps) {
    case 2: return whole(std::integral_constant<int, 2>{});
    case 3: return whole(std::integral_constant<int, 3>{});
    default: return whole(std::integral_constant<int, 4>{});
  }
}

int check(const morph_conv* a, int dtype) {
  if (!a || a->batch < 0 || a->steps < 0 || a->dim < 0) return MORPH_EINVAL;
  if (a->taps < 2 || a->taps > MORPH_CONV_MAX_TAPS) return MORPH_ERANGE;
  if (!known_dtype(dtype) || (a->weight_dtype != MORPH_DTYPE_F32 && a->weight_dtype != dtype)) return MORPH_EDTYPE;
  if (a->batch > 0 && a->dim > 0 && ((a->steps > 0 && !a->x) || !a->weight)) return MORPH_EINVAL;
  const int64_t all = INT64_MAX >> 12;
  if (a->batch > 0 && a->dim > 0 && (a->dim > all / a->batch || a->steps > all / a->batch / a->dim)) return MORPH_ERANGE;
  return MORPH_OK;
}

int64_t over(int64_t n, int64_t by) { return (n + by - 1) / by; }

int64_t back_parts(int64_t batch, int64_t steps) {
  const int64_t units = batch * (steps > 0 ? over(steps, 4 * kBackRun) : 1);
  return units < kParts ? units : kParts;
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" int morph_conv_forward(const morph_conv* a, int dtype, void* y, void* after, void* stream) {
  if (const int rc = check(a, dtype)) return rc;
  if (a->batch == 0 || a->dim == 0) return MORPH_OK;
  if ((a->steps > 0 && !y) || !after) return MORPH_EINVAL;
  return by_dtypes(dtype, a->weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    const ConvGrid g{over(a->dim, 64 * V), a->steps > 0 ? over(a->steps, 4 * kRun) : 1};
    if (!launchable(g.channel_blocks * g.time_blocks * a->batch, 256)) return (int)MORPH_ERANGE;
    return by_form(a->taps, a->dim, [&](auto k, auto whole) {
      hipLaunchKernelGGL((conv_kernel<T, W, decltype(k)::value, decltype(whole)::value>),
                         dim3((unsigned)(g.channel_blocks * g.time_blocks * a->batch)), dim3(256), 0, as_stream(stream), *a,
                         g, y, after);
      return launch_status();
    });
  });
}

extern "C" size_t morph_conv_workspace_bytes(int64_t batch, int64_t steps, int64_t dim, int taps) {
  if (batch < 0 || steps < 0 || dim < 0 || taps < 0) return 0;
  return (size_t)back_parts(batch, steps) * (size_t)(taps + 1) * (size_t)dim * sizeof(float);
}

extern "C" int morph_conv_backward(const morph_conv* a, int dtype, const void* dy, int64_t dy_batch, int64_t dy_step,
                                   const void* dafter, void* dx, void* dweight, void* dbias, void* dbefore,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(a, dtype)) return rc;
  if (a->dim == 0) return MORPH_OK;
  if (!dweight || (a->batch > 0 && a->steps > 0 && (!dy || !dx))) return MORPH_EINVAL;
  const size_t need = morph_conv_workspace_bytes(a->batch, a->steps, a->dim, a->taps);
  if (need > 0 && (!workspace || workspace_bytes < need)) return MORPH_EWORKSPACE;
  const int64_t blocks = over(a->dim, 64 * V), sum_blocks = over(a->dim, 64);
  if (!launchable(blocks, 256) || !launchable(sum_blocks, 1024)) return MORPH_ERANGE;
  const ConvGrid g{blocks, a->steps > 0 ? over(a->steps, 4 * kBackRun) : 1};
  const int parts = (int)back_parts(a->batch, a->steps);
  return by_dtypes(dtype, a->weight_dtype, [&](auto t, auto w) {
    using T = decltype(t);
    using W = decltype(w);
    if (parts > 0) {
      const int rc = by_form(a->taps, a->dim, [&](auto k, auto whole) {
        hipLaunchKernelGGL((conv_back_kernel<T, W, decltype(k)::value, decltype(whole)::value>),
                           dim3((unsigned)blocks, parts), dim3(256), 0, as_stream(stream), *a, g, dy, dy_batch, dy_step,
                           dafter, dx, dbefore, static_cast<float*>(workspace));
        return launch_status();
      });
      if (rc != MORPH_OK) return rc;
    }
    hipLaunchKernelGGL(conv_sum_kernel<W>, dim3((unsigned)sum_blocks, a->taps + 1), dim3(1024), 0, as_stream(stream),
                       static_cast<const float*>(workspace), parts, a->dim, a->taps, dweight, dbias);
    return launch_status();
  });
}
