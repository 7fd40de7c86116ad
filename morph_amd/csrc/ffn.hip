// Gated feed-forward block (morph_layers.h), forward and backward: its products as MFMA
// kernels whose epilogues carry the gate.
//
//   forward   [g u] = x [gate up]^T with h = silu(g) u in the epilogue; y = h down^T
//   backward  dh = dy down with h, dg and du in the epilogue; dx = [dg du] [gate; up];
//             dgate = dg^T x, dup = du^T x, ddown = dy^T h
//
// g and u meet in one workgroup, so neither is written unless the backward needs it, and dh
// never is.  Where 8-bit groups are kept they are made from the FP32 sums in the epilogue.
//
// ffn_any_kernel takes operands of any stride and alignment, any size: 64 x 64 tiles
// through LDS, loaded element by element along whichever index is contiguous.
#include "ffn.h"

namespace morph {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64, kDepth = 32;

template <typename T, FfnEpilogue kE>
__global__ __launch_bounds__(kThreads) void ffn_any_kernel(const FfnProduct a) {
  constexpr int kRow = kDepth + 8;  // LDS row: 80 bytes, 16-byte fragments on distinct banks
  constexpr bool kDual = kE == FfnEpilogue::kGate;
  constexpr int kCols = kDual ? kTile / 2 : kTile;  // columns of the output
  __shared__ __attribute__((aligned(16))) uint16_t sp[kTile][kRow], sq[kTile][kRow];
  __shared__ float sum[kTile][kTile + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kCols;

  f32x16 acc{};
  for (int seg = 0; seg < a.segments; ++seg) {
    for (int64_t k0 = 0; k0 < a.K; k0 += kDepth) {
      auto load = [&](const FfnOperand& o, int64_t row0, int64_t rows, uint16_t (*dst)[kRow], int count) {
#pragma unroll
        for (int i = 0; i < kTile * kDepth / kThreads; ++i) {
          const int x = tid + i * kThreads;
          const int r = o.ks == 1 ? x / kDepth : x % count, k = o.ks == 1 ? x % kDepth : x / count;
          if (r < count && k < kDepth)
            dst[r][k] = row0 + r < rows && k0 + k < a.K ? o.p[(row0 + r) * o.rs + (k0 + k) * o.ks] : 0;
        }
      };
      __syncthreads();
      load(a.P[seg], m0, a.M, sp, kTile);
      if constexpr (kDual) {
        load(a.Q[0], n0, a.N, sq, kCols);
        load(a.Q[1], n0, a.N, sq + kCols, kCols);
      } else {
        load(a.Q[seg], n0, a.N, sq, kTile);
      }
      __syncthreads();
      const int rp = (wave >> 1) * 32 + (lane & 31), rq = (wave & 1) * 32 + (lane & 31);
#pragma unroll
      for (int k = 0; k < kDepth; k += 16) {
        const u32x4 p = *reinterpret_cast<const u32x4*>(&sp[rp][k + 8 * (lane >> 5)]);
        const u32x4 q = *reinterpret_cast<const u32x4*>(&sq[rq][k + 8 * (lane >> 5)]);
        acc = mfma32<T>(p, q, acc);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 16; ++r)
    sum[(wave >> 1) * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)][(wave & 1) * 32 + (lane & 31)] = acc[r];
  __syncthreads();

  // a quad of lanes per row: eight consecutive columns each, so a group of 32 per quad
  const int64_t row = m0 + (tid >> 2);
  if (row >= a.M) return;
  const float* s = sum[tid >> 2];
#pragma unroll
  for (int c0 = 0; c0 < kCols; c0 += 32) {
    const int c = c0 + 8 * (tid & 3);
    if constexpr (kE == FfnEpilogue::kStore) {
      for (int k = 0; k < 8; ++k)
        if (n0 + c + k < a.N) a.C[row * a.ldc + n0 + c + k] = (uint16_t)from_float<T>(s[c + k]);
    } else {
      if (n0 + c0 >= a.ldc) break;  // rows are whole groups; columns behind N are zero
      const int64_t at = row * a.ldc + n0 + c;
      float x[8], g[8], u[8];
      if constexpr (kDual) {
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = s[c + k], u[k] = s[kCols + c + k], x[k] = ffn_gate(g[k], u[k]);
        ffn_keep8(a.keep, a.g, a.g_exponents, at, g);
        ffn_keep8(a.keep, a.u, a.u_exponents, at, u);
      } else {
        ffn_kept8(a.keep, a.g, a.g_exponents, at, g);
        ffn_kept8(a.keep, a.u, a.u_exponents, at, u);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const GateGrad d = ffn_gate_grad(s[c + k], g[k], u[k]);
          x[k] = d.h, g[k] = d.dg, u[k] = d.du;
        }
        *reinterpret_cast<u32x4*>(a.dg + at) = pack8<T>(g);
        *reinterpret_cast<u32x4*>(a.du + at) = pack8<T>(u);
      }
      *reinterpret_cast<u32x4*>(a.C + at) = pack8<T>(x);
    }
  }
}

template <typename T>
int launch_product(FfnEpilogue e, const FfnProduct& a, hipStream_t s) {
  if (a.M == 0 || a.N == 0) return MORPH_OK;
  const int cols = e == FfnEpilogue::kGate ? kTile / 2 : kTile;
  const int64_t gx = (a.N + cols - 1) / cols, gy = (a.M + kTile - 1) / kTile;
  const dim3 grid((unsigned)gx, (unsigned)gy), block(kThreads);
  if (e == FfnEpilogue::kStore)
    hipLaunchKernelGGL((ffn_any_kernel<T, FfnEpilogue::kStore>), grid, block, 0, s, a);
  else if (e == FfnEpilogue::kGate)
    hipLaunchKernelGGL((ffn_any_kernel<T, FfnEpilogue::kGate>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((ffn_any_kernel<T, FfnEpilogue::kGateGrad>), grid, block, 0, s, a);
  return launch_status();
}

int product(int dtype, FfnEpilogue e, const FfnProduct& a, hipStream_t s) {
  return dtype == MORPH_DTYPE_F16 ? launch_product<F16>(e, a, s) : launch_product<BF16>(e, a, s);
}

int64_t whole_groups(int64_t n) { return (n + MORPH_ACT_GROUP - 1) / MORPH_ACT_GROUP * MORPH_ACT_GROUP; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Limits under which every offset fits 64 bits and every grid the hardware (65535 tiles of
// rows in grid.y).
constexpr int64_t kMaxRows = 65535 * (int64_t)kTile, kMaxDim = int64_t(1) << 22;

int ffn_check(const morph_ffn* a, int dtype, const morph_ffn_saved* saved, bool backward) {
  if (a == nullptr || a->rows < 0 || a->d < 1 || a->ff < 1) return MORPH_EINVAL;
  if (dtype != MORPH_DTYPE_F16 && dtype != MORPH_DTYPE_BF16) return MORPH_EDTYPE;
  if (a->rows > kMaxRows || a->d > kMaxDim || a->ff > kMaxDim) return MORPH_ERANGE;
  const int keep = saved ? saved->keep : MORPH_FFN_KEEP_NONE;
  if (keep < MORPH_FFN_KEEP_NONE || keep > MORPH_FFN_KEEP_ACT8 || (backward && keep == MORPH_FFN_KEEP_NONE))
    return MORPH_EINVAL;
  const bool reads_x = a->rows > 0 && !(backward && keep == MORPH_FFN_KEEP_ACT8);
  if ((reads_x && (a->x == nullptr || a->x_ld < a->d)) || a->gate == nullptr || a->up == nullptr ||
      a->down == nullptr || a->gate_ld < a->d || a->up_ld < a->d || a->down_ld < a->ff)
    return MORPH_EINVAL;
  auto odd = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 2 != 0; };
  if ((reads_x && odd(a->x)) || odd(a->gate) || odd(a->up) || odd(a->down)) return MORPH_EINVAL;
  constexpr int64_t kMaxLd = int64_t(1) << 32;
  if ((reads_x && a->x_ld > kMaxLd) || a->gate_ld > kMaxLd || a->up_ld > kMaxLd || a->down_ld > kMaxLd)
    return MORPH_ERANGE;
  if (a->rows == 0 || keep == MORPH_FFN_KEEP_NONE) return MORPH_OK;
  if (saved->gate == nullptr || saved->up == nullptr || !aligned16(saved->gate) || !aligned16(saved->up))
    return MORPH_EINVAL;
  if (keep == MORPH_FFN_KEEP_ACT8 &&
      (saved->gate_exponents == nullptr || saved->up_exponents == nullptr || saved->x_codes == nullptr ||
       saved->x_exponents == nullptr || !aligned16(saved->x_codes)))
    return MORPH_EINVAL;
  return MORPH_OK;
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" size_t morph_ffn_workspace_bytes(int64_t rows, int64_t d, int64_t ff, int keep, int backward) {
  if (rows <= 0 || d <= 0 || ff <= 0) return 0;
  const size_t wide = 2 * (size_t)rows * (size_t)whole_groups(ff);  // h (and dg, du)
  if (!backward) return wide;
  return 3 * wide + (keep == MORPH_FFN_KEEP_ACT8 ? 2 * (size_t)rows * (size_t)whole_groups(d) : 0);
}

extern "C" int morph_ffn_forward(const morph_ffn* a, int dtype, const morph_ffn_saved* saved, void* y,
                                 int64_t y_ld, void* workspace, size_t workspace_bytes, void* stream) {
  int status = ffn_check(a, dtype, saved, false);
  if (status != MORPH_OK) return status;
  if (a->rows == 0) return MORPH_OK;
  if (y == nullptr || y_ld < a->d || reinterpret_cast<uintptr_t>(y) % 2) return MORPH_EINVAL;
  const int keep = saved ? saved->keep : MORPH_FFN_KEEP_NONE;
  if (workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < morph_ffn_workspace_bytes(a->rows, a->d, a->ff, keep, 0))
    return MORPH_EWORKSPACE;
  hipStream_t s = as_stream(stream);
  uint16_t* h = static_cast<uint16_t*>(workspace);
  const int64_t ld = whole_groups(a->ff);
  auto rows16 = [](const void* p, int64_t ldp) {
    return FfnOperand{static_cast<const uint16_t*>(p), ldp, 1};
  };
  if (keep == MORPH_FFN_KEEP_ACT8) {
    status = morph_act_pack(a->x, dtype, a->rows, a->d, a->x_ld, saved->x_codes, saved->x_exponents, stream);
    if (status != MORPH_OK) return status;
  }
  FfnProduct p{};
  p.P[0] = rows16(a->x, a->x_ld);
  p.Q[0] = rows16(a->gate, a->gate_ld);
  p.Q[1] = rows16(a->up, a->up_ld);
  p.M = a->rows, p.N = a->ff, p.K = a->d, p.segments = 1, p.keep = keep;
  p.C = h, p.ldc = ld;
  if (keep != MORPH_FFN_KEEP_NONE)
    p.g = saved->gate, p.u = saved->up, p.g_exponents = saved->gate_exponents, p.u_exponents = saved->up_exponents;
  status = product(dtype, FfnEpilogue::kGate, p, s);
  if (status != MORPH_OK) return status;
  FfnProduct o{};
  o.P[0] = rows16(h, ld);
  o.Q[0] = rows16(a->down, a->down_ld);
  o.M = a->rows, o.N = a->d, o.K = a->ff, o.segments = 1;
  o.C = static_cast<uint16_t*>(y), o.ldc = y_ld;
  return product(dtype, FfnEpilogue::kStore, o, s);
}

extern "C" int morph_ffn_backward(const morph_ffn* a, int dtype, const morph_ffn_saved* saved,
                                  const void* dy, int64_t dy_ld, void* dx, void* dgate, void* dup,
                                  void* ddown, void* workspace, size_t workspace_bytes, void* stream) {
  int status = ffn_check(a, dtype, saved, true);
  if (status != MORPH_OK) return status;
  if (dgate == nullptr || dup == nullptr || ddown == nullptr) return MORPH_EINVAL;
  if (a->rows > 0 && (dy == nullptr || dx == nullptr || dy_ld < a->d || dy_ld > (int64_t(1) << 32)))
    return MORPH_EINVAL;
  if ((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dgate) |
       reinterpret_cast<uintptr_t>(dup) | reinterpret_cast<uintptr_t>(ddown)) % 2)
    return MORPH_EINVAL;
  if (a->rows > 0 && (workspace == nullptr || !aligned16(workspace) ||
                      workspace_bytes < morph_ffn_workspace_bytes(a->rows, a->d, a->ff, saved->keep, 1)))
    return MORPH_EWORKSPACE;
  hipStream_t s = as_stream(stream);
  const int64_t ld = whole_groups(a->ff);
  uint16_t* h = static_cast<uint16_t*>(workspace);
  uint16_t *dg = h + a->rows * ld, *du = dg + a->rows * ld, *xs = du + a->rows * ld;
  const uint16_t* x = static_cast<const uint16_t*>(a->x);
  int64_t x_ld = a->x_ld;
  if (saved->keep == MORPH_FFN_KEEP_ACT8 && a->rows > 0) {
    x = xs, x_ld = whole_groups(a->d);
    status = morph_act_unpack(saved->x_codes, saved->x_exponents, a->rows, a->d, xs, dtype, x_ld, stream);
    if (status != MORPH_OK) return status;
  }
  auto along = [](const void* p, int64_t ldp) {  // the rows of a stored matrix, K along them
    return FfnOperand{static_cast<const uint16_t*>(p), ldp, 1};
  };
  auto across = [](const void* p, int64_t ldp) {  // its columns, K across its rows
    return FfnOperand{static_cast<const uint16_t*>(p), 1, ldp};
  };
  auto run = [&](FfnEpilogue e, const FfnProduct& p) {
    if (status == MORPH_OK) status = product(dtype, e, p, s);
  };
  FfnProduct p{};
  p.P[0] = along(dy, dy_ld), p.Q[0] = across(a->down, a->down_ld);
  p.M = a->rows, p.N = a->ff, p.K = a->d, p.segments = 1, p.keep = saved->keep;
  p.C = h, p.ldc = ld, p.dg = dg, p.du = du;
  p.g = saved->gate, p.u = saved->up, p.g_exponents = saved->gate_exponents, p.u_exponents = saved->up_exponents;
  run(FfnEpilogue::kGateGrad, p);

  FfnProduct q{};
  q.P[0] = along(dg, ld), q.Q[0] = across(a->gate, a->gate_ld);
  q.P[1] = along(du, ld), q.Q[1] = across(a->up, a->up_ld);
  q.M = a->rows, q.N = a->d, q.K = a->ff, q.segments = 2;
  q.C = static_cast<uint16_t*>(dx), q.ldc = a->d;
  run(FfnEpilogue::kStore, q);

  auto weight = [&](FfnOperand left, int64_t m, FfnOperand right, int64_t n, void* out) {
    FfnProduct w{};
    w.P[0] = left, w.Q[0] = right, w.M = m, w.N = n, w.K = a->rows, w.segments = 1;
    w.C = static_cast<uint16_t*>(out), w.ldc = n;
    run(FfnEpilogue::kStore, w);
  };
  weight(across(dg, ld), a->ff, across(x, x_ld), a->d, dgate);
  weight(across(du, ld), a->ff, across(x, x_ld), a->d, dup);
  weight(across(dy, dy_ld), a->d, across(h, ld), a->ff, ddown);
  return status;
}
