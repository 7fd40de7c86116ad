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
// The tiles of ffn_tiles.h take operands whose rows are 16-byte aligned and a multiple of 8
// values long; operands of other widths are copied to such rows first (ffn_pad_kernel: a
// read and a write of them beside the product's many reads).  ffn_any_kernel takes operands of any stride
// and alignment, any size: 64 x 64 tiles through LDS, loaded element by element along whichever index is
// contiguous.  It runs where a width is a multiple of 8 but the address is off 16 bytes or the row stride is no
// multiple of 8, and for dx where gate and up differ in their row strides, and it is slow: 2048 rows of 3072 x 6144
// in BF16 take 4490 us with such a gate (255 with none, 253 with a copy of it ahead of the call), forward and
// backward 8090 (794).
#include <algorithm>
#include <cmath>

#include "ffn_rows.h"
#include "ffn_tiles.h"

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
int launch_any(FfnEpilogue e, const FfnProduct& a, hipStream_t s) {
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

// ---- tiles ----------------------------------------------------------------------

// Time of a launch of `tiles` tiles over kt stages of K, in us: the constants of the
// Newton-Schulz products' launches (gemm.hip), which run the same pipeline, and what the
// gate's epilogues add.  Measured, us with 64 x 64 / 128 x 128 / 256 x 128 / 256 x 256, rows x d x ff:
//   gate: 512 x 3072 x 6144 64 / 49 / 44 / 68, 2048: 282 / 164 / 149 / 158, 4096 (FP32 kept): 557 / 377 / 316 / 270;
//   down: 512 x 3072 x 6144 41 / 61 / 68 / 106, 2048: 150 / 108 / 89 / 120, 4096: 259 / 182 / 179 / 138;
//   gate's gradient: 512 40 / 38 / 49 / 78, 2048: 139 / 98 / 112 / 104, 4096 (FP32 kept): 283 / 224 / 223 / 244;
//   dx: 512 88 / 108 / 143 / 223, 2048: 282 / 197 / 173 / 247, 4096: 551 / 348 / 348 / 285;
//   weights: 512 104 / 76 / 87 / 81, 2048: 360 / 234 / 237 / 219, 4096: 800 / 459 / 458 / 412.
// Other widths, FP16, FP32 kept, 333 x 200 x 536 / 1024 x 768 x 2048 / 512 x 1536 x 4096 / 4096 x 768 x 2048 /
// 2048 x 1408 x 5528 / 4096 x 2048 x 5504, all four shapes of each (K whole): what the rule takes over the best of them:
//   gate: 1.00 / 1.00 / 1.00 / 1.00 / 1.06 / 1.00, nothing kept the same but 1.08 at 2048 x 1408 x 5528;
//   down: 1.00 / 1.00 / 1.00 / 1.00 / 1.00 / 1.11; dx: 1.00 / 1.00 / 1.00 / 1.00 / 1.00 / 1.11;
//   gate's gradient: 1.00 / 1.00 / 1.00 / 1.12 / 1.00 / 1.00; weights: 1.00 / 1.00 / 1.00 / 1.00 / 1.02 / 1.02.
// So 5.9 against 8.6 to 18.1 us for down at 333 x 200 x 536, 101.7 against 158 / 91.9 / 120 at 4096 x 2048 x 5504.
double tiles_us(FfnShape shape, int64_t tiles, int64_t kt, double epilogue) {
  const double q = (double)tiles / 256.0, n = std::ceil(q), full = q / n;
  switch (shape) {
    case kTile256: return n * ((double)kt * (1.0 + 0.45 * full * full) + 8.5 + 4 * epilogue);
    case kTile256x128: return n * ((double)kt * (0.65 + 0.2 * full * full) + 6.0 + 2 * epilogue);
    case kTile128: {
      const double stage = n <= 1.0 ? 0.55 : n <= 2.0 ? 0.8 : n <= 8.0 ? 0.45 * n + 0.1 : 0.5 * n - 0.3;
      return (double)kt * stage + n * (1.3 + epilogue) + 2.0;
    }
    default: return (double)kt * std::max(0.22, 0.24 * q) + (0.2 + 0.1 * epilogue) * q + 3.0;
  }
}

// A product in the tiles' form.  `padded`: of an internal buffer, whose rows hold zeros up to
// a multiple of 32.
struct Side {
  const void* p;
  int64_t ld;
  bool padded;
};
bool fits(const Side& s, int64_t width) {
  return reinterpret_cast<uintptr_t>(s.p) % 16 == 0 && s.ld % 8 == 0 && s.ld <= (int64_t(1) << 22) &&
         (width % 8 == 0 || s.padded);
}

// The most parts of K that tiles of `edge` of an output M x N of kt stages are split into: no more than two
// workgroups per CU, and eight stages, twice a tile's start, in each.  Measured, us, whole in the best tiles / in
// parts with the launch that joins them, as choose() takes them: forward of 100 rows of 3072 x 6144 72 / 53 (128 x 128,
// 8 parts), 256 84 / 75 (128, 4), 512 104 / 94 (128, 4), 1024 146 / 138 (128, 2), 256 rows of 640 x 2336 24 / 21 (64, 4),
// dx of 7 rows of 2880 x 6144 70 / 20 (64, 8); left whole: 1413 rows of 1408 x 5528 108 / 117, 2048 of 512 x 2048, forward
// and backward, 103 / 105.
int splits_of(int64_t edge, int64_t M, int64_t N, int64_t kt) {
  const int64_t tiles = ((M + edge - 1) / edge) * ((N + edge - 1) / edge);
  int n = 1;
  while (n < 8 && 2 * n * tiles <= 512 && kt >= 16 * n) n *= 2;
  return n;
}
int64_t parts_bytes(int64_t M, int64_t N, int64_t kt) {
  const int n = std::max(splits_of(64, M, N, kt), splits_of(128, M, N, kt));
  return n > 1 ? 4 * n * M * ((N + 127) / 128 * 128) : 0;
}
int64_t stages(int64_t K) { return (K + 63) / 64; }

// What the sums of a split product's parts cost over one launch's stores, us.
double join_us(int splits, int64_t M, int64_t N) { return 4.0 + (double)splits * (double)(M * N) * 5e-7; }

// C [M, N] = the parts' sums, in order.  A thread takes eight columns.
template <typename T, int kSplits>
__global__ __launch_bounds__(64) void ffn_join_kernel(const float* __restrict__ parts, int64_t M, int64_t N,
                                                      int64_t ld, uint16_t* __restrict__ C, int64_t ldc, int vector) {
  const int64_t row = blockIdx.y, col = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 8;
  if (col >= N) return;
  f32x4 x[kSplits][2];
#pragma unroll
  for (int i = 0; i < kSplits; ++i) {
    const f32x4* at = reinterpret_cast<const f32x4*>(parts + (i * M + row) * ld + col);
    x[i][0] = at[0], x[i][1] = at[1];
  }
  float sum[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    sum[k] = x[0][k >> 2][k & 3];
#pragma unroll
    for (int i = 1; i < kSplits; ++i) sum[k] += x[i][k >> 2][k & 3];
  }
  store_eight(C + row * ldc + col, pack8<T>(sum), N - col, vector != 0);
}

struct Launch {
  FfnTileArgs a{};
  bool ok = true;
  Launch() { a.splits = 1; }
  void add(const Side& p, const Side& q, int64_t p_width, int64_t q_width, int64_t M, int64_t N, void* c,
           int64_t ldc) {
    FfnTileProblem& o = a.p[a.count++];
    o.P[0] = o.P[1] = static_cast<const uint16_t*>(p.p);
    o.Q[0] = o.Q[1] = static_cast<const uint16_t*>(q.p);
    o.ldp[0] = o.ldp[1] = p.ld, o.ldq[0] = o.ldq[1] = q.ld;
    o.C = static_cast<uint16_t*>(c), o.ldc = ldc, o.M = (int32_t)M, o.N = (int32_t)N;
    o.vector = reinterpret_cast<uintptr_t>(c) % 16 == 0 && ldc % 8 == 0;
    ok = ok && fits(p, p_width) && fits(q, q_width);
  }
  // The tiles' shape for this K, and with it the outputs' tiles; split: 2 where a tile has half as
  // many output columns (the gate's).  parts: memory for the sums of K's parts (parts_bytes), which
  // small tiles of one output of `kt` stages may then have.
  FfnShape choose(int64_t K, int split, double epilogue, int64_t kt = 0, void* parts = nullptr) {
    a.K = (int32_t)K;
    if (kt == 0) kt = stages(K);
    auto tiles = [&](int shape) {
      const int tm = kFfnTileM[shape], tn = kFfnTileN[shape] / split;
      int64_t n = 0;
      for (int i = 0; i < a.count; ++i) {
        FfnTileProblem& o = a.p[i];
        o.first = (int32_t)n;
        o.tiles_m = (o.M + tm - 1) / tm, o.tiles_n = (o.N + tn - 1) / tn;
        n += (int64_t)o.tiles_m * o.tiles_n;
      }
      return n;
    };
    int shape = 0;
    double best = 0;
    for (int i = 0; i < kFfnShapes; ++i) {
      const double us = tiles_us((FfnShape)i, tiles(i), kt, epilogue);
      if (i == 0 || us < best) shape = i, best = us;
    }
    const double whole = best;
    for (int i = kTile128; parts != nullptr && i <= kTile64; ++i) {
      const int most = splits_of(kFfnTileM[i], a.p[0].M, a.p[0].N, kt);
      for (int n = 2; n <= most; n *= 2) {
        const double us = tiles_us((FfnShape)i, n * tiles(i), (kt + n - 1) / n, epilogue) + join_us(n, a.p[0].M, a.p[0].N);
        if (us < 0.95 * whole && us < best) shape = i, best = us, a.splits = n;
      }
    }
    if (a.splits > 1) a.parts = static_cast<float*>(parts);
    const int64_t n = tiles(shape);
    ok = ok && launchable(n + 7, kFfnThreads);
    a.total = (int32_t)n;
    return (FfnShape)shape;
  }
  unsigned grid() const { return (unsigned)((a.total + 7) / 8 * 8); }
  // Behind a launch: the sums of its parts, if it has some.
  int join(FfnShape shape, int dtype, hipStream_t s) const {
    const int status = launch_status();
    if (status != MORPH_OK || a.splits == 1) return status;
    const FfnTileProblem& o = a.p[0];
    const int tile_n = kFfnTileN[shape];
    const dim3 grid((unsigned)((o.N + 511) / 512), (unsigned)o.M);
    auto with = [&](auto type, auto splits) {
      hipLaunchKernelGGL((ffn_join_kernel<decltype(type), decltype(splits)::value>), grid, dim3(64), 0, s, a.parts,
                         (int64_t)o.M, (int64_t)o.N, (int64_t)o.tiles_n * tile_n, o.C, o.ldc, (int)o.vector);
    };
    auto typed = [&](auto type) {
      if (a.splits == 2) with(type, std::integral_constant<int, 2>{});
      else if (a.splits == 4) with(type, std::integral_constant<int, 4>{});
      else with(type, std::integral_constant<int, 8>{});
    };
    if (dtype == MORPH_DTYPE_F16) typed(F16{});
    else typed(BF16{});
    return launch_status();
  }
};

// Up to five matrices copied to rows of whole 16-byte chunks, zero behind their width: a wave
// per row, so that no thread divides to find its place.  Three weights of 2586 x 5905 (184 MB read and
// written) in 29 us; a thread per chunk that it loaded value by value took 70.
struct PadMatrix {
  const uint16_t* src;
  uint16_t* dst;
  int64_t cols, src_ld, dst_ld, first;  // first: its first row of the launch
};
struct PadArgs {
  PadMatrix m[5];
  int64_t rows;
  int32_t count;
};
__global__ __launch_bounds__(kThreads) void ffn_pad_kernel(const PadArgs a) {
  const int64_t at = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (at >= a.rows) return;
  int i = 0;
  while (i + 1 < a.count && at >= a.m[i + 1].first) ++i;
  const PadMatrix& m = a.m[i];
  const int64_t row = at - m.first;
  const uint16_t* src = m.src + row * m.src_ld;
  uint16_t* dst = m.dst + row * m.dst_ld;
  const int64_t whole = m.cols / 8;
#pragma unroll 4
  for (int64_t c = threadIdx.x & 63; c < whole; c += 64) *reinterpret_cast<u32x4*>(dst + 8 * c) = load_eight(src + 8 * c);
  if ((threadIdx.x & 63) < 8) {  // the chunk that is not whole
    const int64_t k = 8 * whole + (threadIdx.x & 63);
    dst[k] = k < m.cols ? src[k] : (uint16_t)0;
  }
}

int64_t padded_bytes(int64_t rows, int64_t cols) { return rows * ((cols + 7) / 8 * 8) * 2; }

// Copies the sides whose width is no multiple of 8 into `room` (16-byte aligned, as much as
// padded_bytes says of each) and points them there.
struct Padding {
  PadArgs a{};
  char* room;
  explicit Padding(void* p) : room(static_cast<char*>(p)) {}
  void add(Side& s, int64_t rows, int64_t cols) {
    if (cols % 8 == 0 || rows == 0) return;
    PadMatrix& m = a.m[a.count++];
    m = PadMatrix{static_cast<const uint16_t*>(s.p), reinterpret_cast<uint16_t*>(room), cols, s.ld,
                  (cols + 7) / 8 * 8, a.rows};
    a.rows += rows;
    room += padded_bytes(rows, cols);
    s = Side{m.dst, m.dst_ld, true};
  }
  int launch(hipStream_t s) {
    if (a.count == 0) return MORPH_OK;
    const int64_t grid = (a.rows + kThreads / 64 - 1) / (kThreads / 64);
    if (!launchable(grid, kThreads)) return MORPH_ERANGE;
    hipLaunchKernelGGL(ffn_pad_kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, a);
    return launch_status();
  }
};

// Whether a forward's products take the few-rows kernels, which read any alignment (down for 7 rows
// of 2880 x 6144: 14 us, 64 x 64 tiles 36); the gate's keeps nothing.
bool few_down(int64_t rows) { return rows <= kFewRows; }
bool few_gate(int64_t rows, int keep) { return rows <= kFewRows && keep == MORPH_FFN_KEEP_NONE; }

int64_t whole_groups(int64_t n) { return (n + MORPH_ACT_GROUP - 1) / MORPH_ACT_GROUP * MORPH_ACT_GROUP; }

int any(int dtype, FfnEpilogue e, const FfnProduct& a, hipStream_t s) {
  return dtype == MORPH_DTYPE_F16 ? launch_any<F16>(e, a, s) : launch_any<BF16>(e, a, s);
}
const uint16_t* u16(const Side& s) { return static_cast<const uint16_t*>(s.p); }
FfnOperand along(const Side& s) { return FfnOperand{static_cast<const uint16_t*>(s.p), s.ld, 1}; }
FfnOperand across(const Side& s) { return FfnOperand{static_cast<const uint16_t*>(s.p), 1, s.ld}; }

// h (row length ld) and what `saved` keeps, from x.
int gate_product(int dtype, const Side& x, const Side& gate, const Side& up, int64_t rows, int64_t d, int64_t ff,
                 const morph_ffn_saved* saved, uint16_t* h, int64_t ld, hipStream_t s) {
  const int keep = saved ? saved->keep : MORPH_FFN_KEEP_NONE;
  // The few-rows kernel reads P's fragments from memory for every weight row's: past 32 rows
  // the tiles are faster where they fit (33 to 64 rows of 3072 x 6144: 37 against 26 us).
  if (few_gate(rows, keep) && (rows <= 32 || !(fits(x, d) && fits(gate, d) && fits(up, d))))
    return ffn_few_rows(dtype, true, u16(x), x.ld, u16(gate), gate.ld, u16(up), up.ld, rows, ff, d, h, ld, s);
  Launch l;
  l.add(x, gate, d, d, rows, ff, h, ld);
  l.ok = l.ok && fits(up, d);
  l.a.p[0].Q[1] = static_cast<const uint16_t*>(up.p), l.a.p[0].ldq[1] = up.ld;
  const FfnShape shape = l.choose(d, 2, keep == MORPH_FFN_KEEP_NONE ? 0.0 : 1.0);
  if (keep != MORPH_FFN_KEEP_NONE)
    l.a.g = saved->gate, l.a.u = saved->up, l.a.g_exponents = saved->gate_exponents,
    l.a.u_exponents = saved->up_exponents;
  if (l.ok) {
    ffn_tile_gate(shape, dtype, keep, l.grid(), s, l.a);
    return launch_status();
  }
  FfnProduct p{};
  p.P[0] = along(x), p.Q[0] = along(gate), p.Q[1] = along(up);
  p.M = rows, p.N = ff, p.K = d, p.segments = 1, p.keep = keep, p.C = h, p.ldc = ld;
  p.g = l.a.g, p.u = l.a.u, p.g_exponents = l.a.g_exponents, p.u_exponents = l.a.u_exponents;
  return any(dtype, FfnEpilogue::kGate, p, s);
}

// y = h down^T.
int down_product(int dtype, const Side& h, const Side& down, int64_t rows, int64_t d, int64_t ff, void* y,
                 int64_t y_ld, void* parts, hipStream_t s) {
  if (few_down(rows))
    return ffn_few_rows(dtype, false, u16(h), h.ld, u16(down), down.ld, nullptr, 0, rows, d, ff,
                        static_cast<uint16_t*>(y), y_ld, s);
  Launch l;
  l.add(h, down, ff, ff, rows, d, y, y_ld);
  const FfnShape shape = l.choose(ff, 1, 0.0, stages(ff), parts);
  if (l.ok) {
    ffn_tile_rows(shape, dtype, l.grid(), s, l.a);
    return l.join(shape, dtype, s);
  }
  FfnProduct p{};
  p.P[0] = along(h), p.Q[0] = along(down);
  p.M = rows, p.N = d, p.K = ff, p.segments = 1, p.C = static_cast<uint16_t*>(y), p.ldc = y_ld;
  return any(dtype, FfnEpilogue::kStore, p, s);
}

// h, dg and du (row length ld) from dy and what was kept.
int grad_product(int dtype, const Side& dy, const Side& down, int64_t rows, int64_t d, int64_t ff,
                 const morph_ffn_saved* saved, uint16_t* h, uint16_t* dg, uint16_t* du, int64_t ld, hipStream_t s) {
  Launch l;
  l.add(dy, down, d, ff, rows, ff, h, ld);
  const FfnShape shape = l.choose(d, 1, saved->keep == MORPH_FFN_KEEP_FULL ? 12.0 : 7.0);
  l.a.dg = dg, l.a.du = du, l.a.g = saved->gate, l.a.u = saved->up;
  l.a.g_exponents = saved->gate_exponents, l.a.u_exponents = saved->up_exponents;
  if (l.ok) {
    ffn_tile_grad(shape, dtype, saved->keep, l.grid(), s, l.a);
    return launch_status();
  }
  FfnProduct p{};
  p.P[0] = along(dy), p.Q[0] = across(down);
  p.M = rows, p.N = ff, p.K = d, p.segments = 1, p.keep = saved->keep, p.C = h, p.ldc = ld, p.dg = dg, p.du = du;
  p.g = saved->gate, p.u = saved->up, p.g_exponents = saved->gate_exponents, p.u_exponents = saved->up_exponents;
  return any(dtype, FfnEpilogue::kGateGrad, p, s);
}

// dx = dg gate + du up.
int input_product(int dtype, const Side& dg, const Side& du, const Side& gate, const Side& up, int64_t rows,
                  int64_t d, int64_t ff, void* dx, void* parts, hipStream_t s) {
  Launch l;
  l.add(dg, gate, ff, d, rows, d, dx, d);
  l.ok = l.ok && fits(up, d) && gate.ld == up.ld;  // one set of offsets for both segments
  FfnTileProblem& o = l.a.p[0];
  o.P[1] = static_cast<const uint16_t*>(du.p), o.Q[1] = static_cast<const uint16_t*>(up.p);
  const FfnShape shape = l.choose(ff, 1, 0.0, 2 * stages(ff), parts);
  if (l.ok) {
    ffn_tile_two(shape, dtype, l.grid(), s, l.a);
    return l.join(shape, dtype, s);
  }
  FfnProduct p{};
  p.P[0] = along(dg), p.Q[0] = across(gate), p.P[1] = along(du), p.Q[1] = across(up);
  p.M = rows, p.N = d, p.K = ff, p.segments = 2, p.C = static_cast<uint16_t*>(dx), p.ldc = d;
  return any(dtype, FfnEpilogue::kStore, p, s);
}

// The three weight gradients, in one launch where the tiles take them.
int weight_products(int dtype, const Side& dg, const Side& du, const Side& x, const Side& dy, const Side& h,
                    int64_t rows, int64_t d, int64_t ff, void* dgate, void* dup, void* ddown, hipStream_t s) {
  struct {
    const Side &p, &q;
    int64_t M, N;
    void* out;
  } w[3] = {{dg, x, ff, d, dgate}, {du, x, ff, d, dup}, {dy, h, d, ff, ddown}};
  Launch l;
  for (auto& e : w) l.add(e.p, e.q, e.M, e.N, e.M, e.N, e.out, e.N);
  const FfnShape shape = l.choose(rows, 1, 0.0);
  if (l.ok && rows > 0) {
    ffn_tile_weights(shape, dtype, l.grid(), s, l.a);
    return launch_status();
  }
  for (auto& e : w) {
    FfnProduct p{};
    p.P[0] = across(e.p), p.Q[0] = across(e.q);
    p.M = e.M, p.N = e.N, p.K = rows, p.segments = 1, p.C = static_cast<uint16_t*>(e.out), p.ldc = e.N;
    const int status = any(dtype, FfnEpilogue::kStore, p, s);
    if (status != MORPH_OK) return status;
  }
  return MORPH_OK;
}

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
  size_t bytes = 2 * (size_t)rows * (size_t)whole_groups(ff);  // h
  if (backward) bytes *= 3;                                     // and dg, du
  if (backward && keep == MORPH_FFN_KEEP_ACT8) bytes += 2 * (size_t)rows * (size_t)whole_groups(d);  // x
  // copies of operands of odd widths
  if (d % 8 && (backward || !few_gate(rows, keep)))
    bytes += (size_t)(padded_bytes(rows, d) * (backward ? 2 : 1) + 2 * padded_bytes(ff, d));
  if (ff % 8 && (backward || !few_down(rows))) bytes += (size_t)padded_bytes(d, ff);
  if (backward || !few_down(rows)) bytes += (size_t)parts_bytes(rows, d, (backward ? 2 : 1) * stages(ff));
  return bytes;
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
  if (keep == MORPH_FFN_KEEP_ACT8) {
    status = morph_act_pack(a->x, dtype, a->rows, a->d, a->x_ld, saved->x_codes, saved->x_exponents, stream);
    if (status != MORPH_OK) return status;
  }
  Side x{a->x, a->x_ld, false}, gate{a->gate, a->gate_ld, false}, up{a->up, a->up_ld, false};
  Side down{a->down, a->down_ld, false};
  Padding pad(h + a->rows * ld);
  if (!few_gate(a->rows, keep)) {
    pad.add(x, a->rows, a->d);
    pad.add(gate, a->ff, a->d);
    pad.add(up, a->ff, a->d);
  }
  if (!few_down(a->rows)) pad.add(down, a->d, a->ff);
  status = pad.launch(s);
  if (status != MORPH_OK) return status;
  status = gate_product(dtype, x, gate, up, a->rows, a->d, a->ff, saved, h, ld, s);
  if (status != MORPH_OK) return status;
  return down_product(dtype, Side{h, ld, true}, down, a->rows, a->d, a->ff, y, y_ld, pad.room, s);
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
  uint16_t *dg = h + a->rows * ld, *du = dg + a->rows * ld, *xs = du + a->rows * ld;  // xs: what else is needed
  Side x{a->x, a->x_ld, false}, gate{a->gate, a->gate_ld, false}, up{a->up, a->up_ld, false};
  Side down{a->down, a->down_ld, false}, sy{dy, dy_ld, false};
  Padding pad(xs);
  if (a->rows > 0) {
    if (saved->keep == MORPH_FFN_KEEP_ACT8) {
      x = Side{xs, whole_groups(a->d), true};
      pad.room += 2 * a->rows * x.ld;
      status = morph_act_unpack(saved->x_codes, saved->x_exponents, a->rows, a->d, xs, dtype | MORPH_ACT_SATURATE,
                                x.ld, stream);
      if (status != MORPH_OK) return status;
    } else {
      pad.add(x, a->rows, a->d);
    }
    pad.add(sy, a->rows, a->d);
    pad.add(gate, a->ff, a->d);
    pad.add(up, a->ff, a->d);
    pad.add(down, a->d, a->ff);
    status = pad.launch(s);
    if (status != MORPH_OK) return status;
  }
  const Side sh{h, ld, true}, sg{dg, ld, true}, su{du, ld, true};
  if (a->rows > 0) {
    status = grad_product(dtype, sy, down, a->rows, a->d, a->ff, saved, h, dg, du, ld, s);
    if (status == MORPH_OK) status = input_product(dtype, sg, su, gate, up, a->rows, a->d, a->ff, dx, pad.room, s);
  }
  if (status == MORPH_OK)
    status = weight_products(dtype, sg, su, x, sy, sh, a->rows, a->d, a->ff, dgate, dup, ddown, s);
  return status;
}
