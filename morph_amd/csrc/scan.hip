// Gated linear recurrence (morph_layers.h) and its backward pass: s_t = a_t s_(t-1) + (1 - a_t) v_t
// along the steps of [batch, steps, dim], every channel on its own.
//
// A lane walks the steps of one channel.  The backward walks the spans of MORPH_SCAN_SPAN steps
// from the last to the first and computes each span's states again from the one that the
// forward kept.
#include <type_traits>

#include "layers.h"

namespace morph {
namespace {

constexpr int kSpan = MORPH_SCAN_SPAN;

template <typename T>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (std::is_same_v<T, F32>)
    return static_cast<const float*>(p)[i];
  else
    return to_float<T>(static_cast<const uint16_t*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void store1(void* p, int64_t i, float x) {
  if constexpr (std::is_same_v<T, F32>)
    static_cast<float*>(p)[i] = x;
  else
    static_cast<uint16_t*>(p)[i] = (uint16_t)from_float<T>(x);
}

template <typename T>
__global__ __launch_bounds__(64) void scan_walk_kernel(morph_scan a, void* __restrict__ y,
                                                       float* __restrict__ last,
                                                       float* __restrict__ states) {
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= a.dim) return;
  float s = a.s0 ? a.s0[b * a.dim + c] : 0.0f;
  const int64_t spans = (a.steps + kSpan - 1) / kSpan;
  for (int64_t t = 0; t < a.steps; ++t) {
    if (states && t % kSpan == 0) states[(b * spans + t / kSpan) * a.dim + c] = s;
    const Sigmoid g = sigmoid(load1<T>(a.f, b * a.f_batch + t * a.f_step + c));
    s = __fmaf_rn(g.a, s, g.b * load1<T>(a.v, b * a.v_batch + t * a.v_step + c));
    float out = s;
    if (a.z) {
      const float z = load1<T>(a.z, b * a.z_batch + t * a.z_step + c);
      out = s * (z * sigmoid(z).a);
    }
    store1<T>(y, (b * a.steps + t) * a.dim + c, out);
  }
  if (last) last[b * a.dim + c] = s;
}

template <typename T>
__global__ __launch_bounds__(64) void scan_walk_back_kernel(morph_scan a, const float* __restrict__ states,
                                                            const void* __restrict__ dy, int64_t dy_batch,
                                                            int64_t dy_step, const float* __restrict__ dlast,
                                                            void* __restrict__ df, void* __restrict__ dv,
                                                            void* __restrict__ dz, float* __restrict__ ds0) {
  __shared__ float before[kSpan][64];  // the state before each step of the span, a column per lane
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
  if (c >= a.dim) return;
  const int lane = threadIdx.x;
  const int64_t spans = (a.steps + kSpan - 1) / kSpan;
  float r = dlast ? dlast[b * a.dim + c] : 0.0f;  // a_(t+1) r_(t+1)
  for (int64_t k = spans - 1; k >= 0; --k) {
    const int64_t t0 = k * kSpan;
    const int n = (int)(a.steps - t0 < kSpan ? a.steps - t0 : kSpan);
    float s = states[(b * spans + k) * a.dim + c];
    for (int i = 0; i < n; ++i) {
      before[i][lane] = s;
      const Sigmoid g = sigmoid(load1<T>(a.f, b * a.f_batch + (t0 + i) * a.f_step + c));
      s = __fmaf_rn(g.a, s, g.b * load1<T>(a.v, b * a.v_batch + (t0 + i) * a.v_step + c));
    }
    for (int i = n - 1; i >= 0; --i) {
      const int64_t t = t0 + i, at = (b * a.steps + t) * a.dim + c;
      const Sigmoid g = sigmoid(load1<T>(a.f, b * a.f_batch + t * a.f_step + c));
      const float v = load1<T>(a.v, b * a.v_batch + t * a.v_step + c);
      float w = load1<T>(dy, b * dy_batch + t * dy_step + c);
      const float prev = before[i][lane];
      if (a.z) {
        const float z = load1<T>(a.z, b * a.z_batch + t * a.z_step + c);
        const Sigmoid q = sigmoid(z);
        const float now = __fmaf_rn(g.a, prev, g.b * v);
        store1<T>(dz, at, w * now * (q.a * __fmaf_rn(z, q.b, 1.0f)));
        w *= z * q.a;
      }
      r += w;
      store1<T>(dv, at, g.b * r);
      store1<T>(df, at, r * (prev - v) * (g.a * g.b));
      r *= g.a;
    }
  }
  if (ds0) ds0[b * a.dim + c] = r;
}

bool float_type(int dtype) {
  return dtype == MORPH_DTYPE_F32 || dtype == MORPH_DTYPE_F16 || dtype == MORPH_DTYPE_BF16;
}

int scan_check(const morph_scan* a, int dtype) {
  if (a == nullptr || a->batch < 0 || a->steps < 0 || a->dim < 0) return MORPH_EINVAL;
  if (!float_type(dtype)) return MORPH_EDTYPE;
  if (a->batch > 65535 || a->dim > (int64_t(1) << 30) || a->steps > (int64_t(1) << 40))
    return MORPH_ERANGE;
  if (a->batch && a->steps && a->dim && (a->f == nullptr || a->v == nullptr)) return MORPH_EINVAL;
  return MORPH_OK;
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" size_t morph_scan_workspace_bytes(int64_t, int64_t, int64_t, int, int) { return 0; }

extern "C" int morph_scan_forward(const morph_scan* scan, int dtype, void* y, float* last,
                                  float* states, void*, size_t, void* stream) {
  const int status = scan_check(scan, dtype);
  if (status != MORPH_OK) return status;
  if (scan->batch == 0 || scan->dim == 0) return MORPH_OK;
  if (scan->steps > 0 && y == nullptr) return MORPH_EINVAL;
  const dim3 grid((unsigned)((scan->dim + 63) / 64), (unsigned)scan->batch);
  hipStream_t s = as_stream(stream);
  if (dtype == MORPH_DTYPE_F32)
    hipLaunchKernelGGL(scan_walk_kernel<F32>, grid, dim3(64), 0, s, *scan, y, last, states);
  else if (dtype == MORPH_DTYPE_F16)
    hipLaunchKernelGGL(scan_walk_kernel<F16>, grid, dim3(64), 0, s, *scan, y, last, states);
  else
    hipLaunchKernelGGL(scan_walk_kernel<BF16>, grid, dim3(64), 0, s, *scan, y, last, states);
  return launch_status();
}

extern "C" int morph_scan_backward(const morph_scan* scan, int dtype, const float* states,
                                   const void* dy, int64_t dy_batch, int64_t dy_step,
                                   const float* dlast, void* df, void* dv, void* dz, float* ds0,
                                   void*, size_t, void* stream) {
  const int status = scan_check(scan, dtype);
  if (status != MORPH_OK) return status;
  if (scan->batch == 0 || scan->dim == 0) return MORPH_OK;
  if (scan->steps > 0 && (states == nullptr || dy == nullptr || df == nullptr || dv == nullptr ||
                          (scan->z != nullptr && dz == nullptr)))
    return MORPH_EINVAL;
  const dim3 grid((unsigned)((scan->dim + 63) / 64), (unsigned)scan->batch);
  hipStream_t s = as_stream(stream);
  if (dtype == MORPH_DTYPE_F32)
    hipLaunchKernelGGL(scan_walk_back_kernel<F32>, grid, dim3(64), 0, s, *scan, states, dy, dy_batch,
                       dy_step, dlast, df, dv, dz, ds0);
  else if (dtype == MORPH_DTYPE_F16)
    hipLaunchKernelGGL(scan_walk_back_kernel<F16>, grid, dim3(64), 0, s, *scan, states, dy, dy_batch,
                       dy_step, dlast, df, dv, dz, ds0);
  else
    hipLaunchKernelGGL(scan_walk_back_kernel<BF16>, grid, dim3(64), 0, s, *scan, states, dy, dy_batch,
                       dy_step, dlast, df, dv, dz, ds0);
  return launch_status();
}
