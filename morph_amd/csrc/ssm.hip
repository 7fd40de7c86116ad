// Selective state space scan (morph_state_space.h) and its backward pass: h_t = exp(d_t A) h_(t-1) + d_t x_t B_t for
// every state of every channel, y = C_t . h_t + skip x, along the steps.
//
// A step costs each state an exponential (a quarter-rate instruction, as long as four others) and four to seven more
// instructions, so with 16 states a channel arithmetic bounds the scan, three times above what HBM does; the layout
// is for that.  A lane has four states of a channel, kLanes neighbouring lanes the channel, a wave 64 / kLanes
// channels and kT consecutive steps.  What belongs to a channel and step alone (softplus, the gate, conversions) is
// done once, by one of its lanes, and spread by DPP; what belongs to a state and step alone (B and C) lies
// converted in LDS.
//
// A workgroup's kW waves take consecutive stretches of a tile of kW kT steps: each walks its stretch from a zero
// state and keeps the states and the products of the gates, the stretches' ends are joined through LDS, and every
// state is then one multiply-add from its true value, without a second exponential.  The workgroup walks the tiles
// in time and carries the state, so nothing waits between workgroups.
//
// The backward walks the tiles from the last to the first.  A tile's entering state was kept by the forward; its
// states come again as there, and the gradient r_t of a state, the same recurrence in reversed time with the
// same gates, is joined across the waves in the same step.  The sums over channels (dB, dC) go through the wave by
// lane swaps, stay in registers over the workgroup's channel groups, and are added up over the workgroups by a
// second launch; the sums over steps (dA, dskip, ddt_bias) stay with the lane and are joined at the end.
// No atomics: a call gives the same bits each time.
#include "stage.h"

namespace morph {
namespace {

constexpr int kT = 8;  // steps of a wave
constexpr int kW = 8;  // waves
static_assert(kT * kW == MORPH_SSM_SPAN, "a backward tile begins with a kept state");
constexpr float kLog2e = 1.44269504088896341f;
constexpr int kMostGroups = 4;     // channel groups of a backward workgroup
constexpr int kBackBlocks = 512;   // workgroups from which on they get more than one

typedef float Four[4];
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

template <int N, typename F, int... I>
__device__ __forceinline__ void each_step(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
// f(0), f(1), ..: the index is a constant in each, as lane controls must be.
template <int N, typename F>
__device__ __forceinline__ void each_step(F&& f) {
  each_step<N>(f, std::make_integer_sequence<int, N>{});
}

// log(1 + e^x) by log(1 + e) = 2 atanh(e / (2 + e)): relative error 3 2^-24 for every x, where log(1 + e) of a small e
// would keep few digits.
__device__ __forceinline__ float softplus(float x) {
  const float e = __builtin_amdgcn_exp2f(-kLog2e * __builtin_fabsf(x));
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
  float p = __fmaf_rn(q, 1.0f / 13.0f, 1.0f / 11.0f);
  p = __fmaf_rn(p, q, 1.0f / 9.0f);
  p = __fmaf_rn(p, q, 1.0f / 7.0f);
  p = __fmaf_rn(p, q, 1.0f / 5.0f);
  p = __fmaf_rn(p, q, 1.0f / 3.0f);
  p = __fmaf_rn(p, q, 1.0f);
  return __fmaf_rn(2.0f * s, p, x > 0.0f ? x : 0.0f);
}

// The value of lane K of this lane's channel, L lanes a channel.
template <int L, int K>
__device__ __forceinline__ float spread(float x) {
  if constexpr (L == 1) return x;
  else if constexpr (L == 2) return dpp<K | K << 2 | (2 + K) << 4 | (2 + K) << 6>(x);
  else if constexpr (L == 4) return dpp<K * 0x55>(x);
  else  // lane (l & ~(L - 1)) | K of 32
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), (0x1F & ~(L - 1)) | K << 5));
}
// The sum over a channel's lanes, in each.
template <int L>
__device__ __forceinline__ float channel_sum(float x) {
  if constexpr (L >= 2) x += dpp<0xB1>(x);    // quad_perm [1,0,3,2]
  if constexpr (L >= 4) x += dpp<0x4E>(x);    // quad_perm [2,3,0,1]
  if constexpr (L >= 8) x += dpp<0x141>(x);   // row_half_mirror
  if constexpr (L >= 16) x += dpp<0x140>(x);  // row_mirror
  return x;
}

__device__ __forceinline__ void swap32(float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
  a = __builtin_bit_cast(float, (uint32_t)r[0]), b = __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ void swap16(float& a, float& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
  a = __builtin_bit_cast(float, (uint32_t)r[0]), b = __builtin_bit_cast(float, (uint32_t)r[1]);
}

// Four states from `first` on of a row of n: one access where rows are whole ones.
__device__ __forceinline__ void load_states(const float* row, int first, int n, Four& x) {
  if (n % 4 == 0) {
    if (first < n) {
      const f32x4 v = *reinterpret_cast<const f32x4_any*>(row + first);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      x[0] = x[1] = x[2] = x[3] = 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = first + j < n ? row[first + j] : 0.0f;
  }
}
__device__ __forceinline__ void store_states(float* row, int first, int n, const Four& x) {
  if (n % 4 == 0) {
    if (first < n) *reinterpret_cast<f32x4_any*>(row + first) = f32x4{x[0], x[1], x[2], x[3]};
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (first + j < n) row[first + j] = x[j];
  }
}

__device__ __forceinline__ f32x4 as_vector(const Four& x) { return f32x4{x[0], x[1], x[2], x[3]}; }

// What one wave wrote to LDS it reads in order; this keeps the compiler to that order.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename T>
struct Bits {
  typedef std::conditional_t<std::is_same_v<T, F32>, uint32_t, uint16_t> type;
};
// A value as loaded, 0 where there is none.
template <typename T>
__device__ __forceinline__ uint32_t load_bits(const void* p, int64_t at, bool there) {
  return there ? (uint32_t)static_cast<const typename Bits<T>::type*>(p)[at] : 0u;
}
template <typename T>
__device__ __forceinline__ float bits_value(uint32_t w) {
  if constexpr (std::is_same_v<T, F32>) return __builtin_bit_cast(float, w);
  else return to_float<T>(w);
}

// A lane's place: its channel, states and, of a wave's kT steps, those whose per-channel work it does.
template <int L>
struct Lane {
  static constexpr int kR = L <= kT ? kT / L : 1;  // steps of each lane: own + i L
  int64_t b, ch;
  int own, first, wave;
  bool active;
  __device__ __forceinline__ Lane(int64_t sequence, int64_t group, int64_t dim) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    own = lane % L, first = own * 4;
    b = sequence, ch = group * (64 / L) + lane / L;
    active = ch < dim;
  }
  __device__ __forceinline__ int64_t step(int64_t t0, int i) const { return t0 + own + i * L; }
  __device__ __forceinline__ bool has(int64_t t, int64_t steps) const { return active && t < steps && own < kT; }
};

// B and C of a wave's steps on their way from memory to its part of LDS, [2][kT][4 L] floats.
template <typename T, int L>
struct Inputs {
  uint32_t w[L];
  __device__ __forceinline__ void fetch(const morph_ssm& a, int64_t b, int64_t t0) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int v = i * 64 + (threadIdx.x & 63), n = v % (4 * L);
      const int64_t t = t0 + v / (4 * L) % kT;
      const bool there = n < a.states && t < a.steps, second = v >= kT * 4 * L;
      w[i] = second ? load_bits<T>(a.C, b * a.C_batch + t * a.C_step + n, there)
                    : load_bits<T>(a.B, b * a.B_batch + t * a.B_step + n, there);
    }
  }
  __device__ __forceinline__ void put(float* to) const {
#pragma unroll
    for (int i = 0; i < L; ++i) to[i * 64 + (threadIdx.x & 63)] = bits_value<T>(w[i]);
  }
};

// Steps of a wave from a zero state: gates a (or their products up to each step), and the states.
template <int L, bool kProducts>
__device__ __forceinline__ void walk(const float (&d)[Lane<L>::kR], const float (&u)[Lane<L>::kR], const Four& A2,
                                     const float* B, int first, Four (&a)[kT], Four (&h)[kT]) {
  each_step<kT>([&](auto step) {
    constexpr int t = decltype(step)::value;
    const float dt = spread<L, t % L>(d[t / L]), ut = spread<L, t % L>(u[t / L]);
    const f32x4 b = *reinterpret_cast<const f32x4*>(B + t * 4 * L + first);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gate = __builtin_amdgcn_exp2f(dt * A2[j]), in = ut * b[j];
      if constexpr (t == 0) {
        a[t][j] = gate, h[t][j] = in;
      } else {
        a[t][j] = kProducts ? gate * a[t - 1][j] : gate;
        h[t][j] = __fmaf_rn(gate, h[t - 1][j], in);
      }
    }
  });
}

template <typename T, int L>
__global__ __launch_bounds__(64 * kW) void ssm_kernel(const morph_ssm a, int64_t groups, void* __restrict__ y,
                                                      float* __restrict__ last, float* __restrict__ kept) {
  constexpr int kR = Lane<L>::kR;
  __shared__ float bc[kW][2 * kT * 4 * L];
  __shared__ f32x4 ends[2][kW][2][64];
  const Lane<L> p(blockIdx.x / groups, blockIdx.x % groups, a.dim);
  const int lane = threadIdx.x & 63;
  const int64_t tiles = (a.steps + kT * kW - 1) / (kT * kW), row = p.b * a.dim + p.ch;
  Four A2 = {}, carry = {};
  float skip = 0.0f, bias = 0.0f;
  if (p.active) {
    load_states(a.A + p.ch * a.states, p.first, a.states, A2);
    if (a.first) load_states(a.first + row * a.states, p.first, a.states, carry);
    if (a.skip) skip = a.skip[p.ch];
    if (a.dt_bias) bias = a.dt_bias[p.ch];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) A2[j] *= kLog2e;

  uint32_t rx[kR], rd[kR], rz[kR];
  Inputs<T, L> in;
  auto fetch = [&](int64_t tile) {
    const int64_t t0 = (tile * kW + p.wave) * kT;
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int64_t t = p.step(t0, i);
      const bool there = p.has(t, a.steps);
      rx[i] = load_bits<T>(a.x, p.b * a.x_batch + t * a.x_step + p.ch, there);
      rd[i] = load_bits<T>(a.dt, p.b * a.dt_batch + t * a.dt_step + p.ch, there);
      rz[i] = a.z ? load_bits<T>(a.z, p.b * a.z_batch + t * a.z_step + p.ch, there) : 0u;
    }
    in.fetch(a, p.b, t0);
  };
  if (tiles > 0) fetch(0);
  for (int64_t tile = 0; tile < tiles; ++tile) {
    const int64_t t0 = (tile * kW + p.wave) * kT;
    float x[kR], d[kR], u[kR], z[kR];
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      x[i] = bits_value<T>(rx[i]);
      z[i] = bits_value<T>(rz[i]);
      d[i] = p.has(p.step(t0, i), a.steps) ? softplus(bits_value<T>(rd[i]) + bias) : 0.0f;
      u[i] = d[i] * x[i];
    }
    float* mine = bc[p.wave];
    in.put(mine);
    wave_order();
    if (tile + 1 < tiles) fetch(tile + 1);
    if (kept && p.wave == 0 && p.active)
      store_states(kept + ((p.b * tiles + tile) * a.dim + p.ch) * a.states, p.first, a.states, carry);
    Four P[kT], h[kT];
    walk<L, true>(d, u, A2, mine, p.first, P, h);
    const int turn = tile & 1;  // every wave has passed the barrier behind the last use of this half
    ends[turn][p.wave][0][lane] = as_vector(P[kT - 1]);
    ends[turn][p.wave][1][lane] = as_vector(h[kT - 1]);
    __syncthreads();
    Four enter;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      if (w == p.wave) {
#pragma unroll
        for (int j = 0; j < 4; ++j) enter[j] = carry[j];
      }
      const f32x4 A = ends[turn][w][0][lane], S = ends[turn][w][1][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) carry[j] = __fmaf_rn(A[j], carry[j], S[j]);
    }
    float out[kR] = {};
    each_step<kT>([&](auto step) {
      constexpr int t = decltype(step)::value;
      const f32x4 c = *reinterpret_cast<const f32x4*>(mine + (kT + t) * 4 * L + p.first);
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) s = __fmaf_rn(c[j], __fmaf_rn(P[t][j], enter[j], h[t][j]), s);
      s = channel_sum<L>(s);
      if (p.own == t % L) out[t / L] = s;
    });
    wave_order();
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      const int64_t t = p.step(t0, i);
      float s = __fmaf_rn(skip, x[i], out[i]);
      if (a.z) s *= z[i] * gate_sigmoid(z[i]);
      if (p.has(t, a.steps)) store_one<T>(y, (p.b * a.steps + t) * a.dim + p.ch, s);
    }
  }
  if (p.wave == 0 && p.active) store_states(last + row * a.states, p.first, a.states, carry);
}

// One step: the state crosses once in and once out, and HBM bounds it.
template <typename T, int L>
__global__ __launch_bounds__(256) void ssm_one_kernel(const morph_ssm a, int64_t groups, void* __restrict__ y,
                                                      float* __restrict__ last, float* __restrict__ kept) {
  const int64_t b = blockIdx.x / groups, lane = threadIdx.x;
  const int64_t ch = (blockIdx.x % groups) * (256 / L) + lane / L;
  const int own = (int)(lane % L), first = own * 4;
  if (ch >= a.dim) return;  // whole channels: their lanes are together
  const int64_t row = b * a.dim + ch;
  Four A, h = {}, B, C;
  if (a.first) load_states(a.first + row * a.states, first, a.states, h);
  load_states(a.A + ch * a.states, first, a.states, A);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool there = first + j < a.states;
    B[j] = bits_value<T>(load_bits<T>(a.B, b * a.B_batch + first + j, there));
    C[j] = bits_value<T>(load_bits<T>(a.C, b * a.C_batch + first + j, there));
  }
  const float x = load_one<T>(a.x, b * a.x_batch + ch), z = a.z ? load_one<T>(a.z, b * a.z_batch + ch) : 0.0f;
  const float d = softplus(load_one<T>(a.dt, b * a.dt_batch + ch) + (a.dt_bias ? a.dt_bias[ch] : 0.0f));
  if (kept) store_states(kept + row * a.states, first, a.states, h);
  const float u = d * x;
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = __fmaf_rn(__builtin_amdgcn_exp2f(d * (A[j] * kLog2e)), h[j], u * B[j]);
    s = __fmaf_rn(C[j], h[j], s);
  }
  store_states(last + row * a.states, first, a.states, h);
  s = channel_sum<L>(s);
  if (own != 0) return;
  if (a.skip) s = __fmaf_rn(a.skip[ch], x, s);
  if (a.z) s *= z * gate_sigmoid(z);
  store_one<T>(y, row, s);
}

// Where a backward's sums lie in its workspace.
struct SsmParts {
  float* bc;       // [blocks of channel groups][batch][steps][2][4 L]: dB, dC
  float* A;        // [batch][dim][states]
  float* skip;     // [batch][dim]
  float* dt_bias;  // [batch][dim]
};

template <typename T, int L>
__global__ __launch_bounds__(64 * kW) void ssm_back_kernel(const morph_ssm a, int64_t blocks, int per,
                                                           const float* __restrict__ kept, const void* __restrict__ dy,
                                                           int64_t dy_batch, int64_t dy_step,
                                                           const float* __restrict__ dlast, const morph_ssm_grads g,
                                                           const SsmParts parts) {
  constexpr int kR = Lane<L>::kR, kRep = 16 / L, kSlots = kRep < kT ? kT / kRep : 1;
  __shared__ float bc[kW][2 * kT * 4 * L];
  __shared__ f32x4 ends[kW][3][64];
  __shared__ f32x4 late[2][kMostGroups][64];           // r behind the tile, times its gate
  __shared__ f32x4 sum_A[kMostGroups][kW][64];         // dA of each wave's steps
  __shared__ float sum_own[kMostGroups][kW][2][64];    // dskip, ddt_bias
  const int64_t b = blockIdx.x / blocks, block = blockIdx.x % blocks, channels = (a.dim + 64 / L - 1) / (64 / L);
  const int count = (int)(channels - block * per < per ? channels - block * per : per);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tiles = (a.steps + kT * kW - 1) / (kT * kW);
  for (int i = 0; i < count; ++i) {
    const Lane<L> p(b, block * per + i, a.dim);
    sum_A[i][wave][lane] = f32x4{0, 0, 0, 0};
    sum_own[i][wave][0][lane] = sum_own[i][wave][1][lane] = 0.0f;
    if (wave == 0) {
      Four r = {};
      if (dlast && p.active) load_states(dlast + (b * a.dim + p.ch) * a.states, p.first, a.states, r);
      late[0][i][lane] = as_vector(r);
    }
  }
  Inputs<T, L> in;
  for (int64_t tile = tiles - 1; tile >= 0; --tile) {
    const int64_t t0 = (tile * kW + wave) * kT;
    const int turn = (int)((tiles - 1 - tile) & 1);
    float* mine = bc[wave];
    in.fetch(a, b, t0);
    in.put(mine);
    wave_order();
    float acc[kSlots][2] = {};
    for (int i = 0; i < count; ++i) {
      const Lane<L> p(b, block * per + i, a.dim);
      float x[kR], d[kR], u[kR], z[kR], e[kR], raw[kR], ds[kR];
      Four A = {}, A2, enter = {};
      float skip = 0.0f, bias = 0.0f;
      if (p.active) {
        load_states(a.A + p.ch * a.states, p.first, a.states, A);
        load_states(kept + ((b * tiles + tile) * a.dim + p.ch) * a.states, p.first, a.states, enter);
        if (a.skip) skip = a.skip[p.ch];
        if (a.dt_bias) bias = a.dt_bias[p.ch];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) A2[j] = A[j] * kLog2e;
#pragma unroll
      for (int k = 0; k < kR; ++k) {
        const int64_t t = p.step(t0, k);
        const bool there = p.has(t, a.steps);
        x[k] = bits_value<T>(load_bits<T>(a.x, b * a.x_batch + t * a.x_step + p.ch, there));
        raw[k] = bits_value<T>(load_bits<T>(a.dt, b * a.dt_batch + t * a.dt_step + p.ch, there)) + bias;
        e[k] = bits_value<T>(load_bits<T>(dy, b * dy_batch + t * dy_step + p.ch, there));
        z[k] = a.z ? bits_value<T>(load_bits<T>(a.z, b * a.z_batch + t * a.z_step + p.ch, there)) : 0.0f;
        d[k] = there ? softplus(raw[k]) : 0.0f;
        u[k] = d[k] * x[k];
        ds[k] = a.z ? e[k] * silu(z[k]).y : e[k];
      }
      Four gate[kT], h[kT];
      walk<L, false>(d, u, A2, mine, p.first, gate, h);
      Four P, Q = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        P[j] = gate[0][j];
#pragma unroll
        for (int t = 1; t < kT; ++t) P[j] *= gate[t][j];
      }
      each_step<kT>([&](auto step) {
        constexpr int t = kT - 1 - decltype(step)::value;
        const float dst = spread<L, t % L>(ds[t / L]);
        const f32x4 c = *reinterpret_cast<const f32x4*>(mine + (kT + t) * 4 * L + p.first);
#pragma unroll
        for (int j = 0; j < 4; ++j) Q[j] = gate[t][j] * __fmaf_rn(c[j], dst, Q[j]);
      });
      ends[wave][0][lane] = as_vector(P);
      ends[wave][1][lane] = as_vector(h[kT - 1]);
      ends[wave][2][lane] = as_vector(Q);
      __syncthreads();
      for (int w = 0; w < wave; ++w) {
        const f32x4 Pw = ends[w][0][lane], S = ends[w][1][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) enter[j] = __fmaf_rn(Pw[j], enter[j], S[j]);
      }
      const f32x4 after = late[turn][i][lane];
      Four r = {after.x, after.y, after.z, after.w};
      for (int w = kW - 1; w > wave; --w) {
        const f32x4 Pw = ends[w][0][lane], Qw = ends[w][2][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __fmaf_rn(Pw[j], r[j], Qw[j]);
      }
      __syncthreads();
      // the states again, from the true one
      each_step<kT>([&](auto step) {
        constexpr int t = decltype(step)::value;
        const float ut = spread<L, t % L>(u[t / L]);
        const f32x4 B = *reinterpret_cast<const f32x4*>(mine + t * 4 * L + p.first);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[t][j] = __fmaf_rn(gate[t][j], t ? h[t ? t - 1 : 0][j] : enter[j], ut * B[j]);
      });
      float rB[kR] = {}, wA[kR] = {}, Ch[kR] = {};
      const f32x4 before = sum_A[i][wave][lane];
      Four dA = {before.x, before.y, before.z, before.w};
      each_step<kT>([&](auto step) {
        constexpr int t = kT - 1 - decltype(step)::value;
        const float dst = spread<L, t % L>(ds[t / L]), dt = spread<L, t % L>(d[t / L]), ut = spread<L, t % L>(u[t / L]);
        const f32x4 B = *reinterpret_cast<const f32x4*>(mine + t * 4 * L + p.first);
        const f32x4 c = *reinterpret_cast<const f32x4*>(mine + (kT + t) * 4 * L + p.first);
        float sB = 0.0f, sA = 0.0f, sC = 0.0f, v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float q = __fmaf_rn(c[j], dst, r[j]);
          sB = __fmaf_rn(q, B[j], sB);
          sC = __fmaf_rn(c[j], h[t][j], sC);
          v[j] = q * ut;
          v[4 + j] = h[t][j] * dst;
          r[j] = gate[t][j] * q;
          const float w = r[j] * (t ? h[t ? t - 1 : 0][j] : enter[j]);
          sA = __fmaf_rn(w, A[j], sA);
          dA[j] = __fmaf_rn(w, dt, dA[j]);
        }
        sB = channel_sum<L>(sB), sA = channel_sum<L>(sA);
        if (p.own == t % L) rB[t / L] = sB, wA[t / L] = sA;
        if (a.z) {
          sC = channel_sum<L>(sC);
          if (p.own == t % L) Ch[t / L] = sC;
        }
        // over the wave's channels: dB to the lower 32 lanes, dC to the upper; states 0 and 1 to even rows of 16
        // lanes, 2 and 3 to odd ones; then within the rows
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          swap32(v[j], v[4 + j]);
          v[j] += v[4 + j];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          swap16(v[j], v[2 + j]);
          v[j] += v[2 + j];
          if constexpr (L <= 8) v[j] += dpp<kRotate8>(v[j]);
          if constexpr (L <= 4) v[j] += dpp<kRotate4>(v[j]);
          if constexpr (L <= 2) v[j] += dpp<kRotate2>(v[j]);
          if constexpr (L <= 1) v[j] += dpp<kRotate1>(v[j]);
          if ((lane & 15) / L == t % kRep) acc[t / kRep][j] += v[j];
        }
      });
      sum_A[i][wave][lane] = as_vector(dA);
      if (wave == 0) late[turn ^ 1][i][lane] = as_vector(r);
      float dskip = 0.0f, dbias = 0.0f;
#pragma unroll
      for (int k = 0; k < kR; ++k) {
        const int64_t t = p.step(t0, k);
        if (!p.has(t, a.steps)) continue;
        const int64_t at = (b * a.steps + t) * a.dim + p.ch;
        const float ddt = __fmaf_rn(x[k], rB[k], wA[k]) * sigmoid(raw[k]).a;
        store_one<T>(g.dx, at, __fmaf_rn(d[k], rB[k], skip * ds[k]));
        store_one<T>(g.ddt, at, ddt);
        if (a.z) store_one<T>(g.dz, at, e[k] * __fmaf_rn(skip, x[k], Ch[k]) * silu(z[k]).slope);
        dskip = __fmaf_rn(ds[k], x[k], dskip);
        dbias += ddt;
      }
      sum_own[i][wave][0][lane] += dskip;
      sum_own[i][wave][1][lane] += dbias;
    }
    wave_order();
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      const int t = s * kRep + (lane & 15) / L;
      if (t < kT && t0 + t < a.steps) {
        float* to = parts.bc + (((block * a.batch + b) * a.steps + t0 + t) * 2 + (lane >> 5)) * 4 * L +
                    (lane & (L - 1)) * 4 + ((lane >> 4) & 1) * 2;
        *reinterpret_cast<f32x2*>(to) = f32x2{acc[s][0], acc[s][1]};
      }
    }
  }
  __syncthreads();
  for (int i = wave; i < count; i += kW) {  // a wave a channel group
    const Lane<L> p(b, block * per + i, a.dim);
    f32x4 dA = sum_A[i][0][lane];
    float own[2] = {sum_own[i][0][0][lane], sum_own[i][0][1][lane]};
#pragma unroll
    for (int w = 1; w < kW; ++w) {
      dA += sum_A[i][w][lane];
      own[0] += sum_own[i][w][0][lane], own[1] += sum_own[i][w][1][lane];
    }
    own[0] = channel_sum<L>(own[0]), own[1] = channel_sum<L>(own[1]);
    if (!p.active) continue;
    const int64_t row = b * a.dim + p.ch;
    const Four sum = {dA.x, dA.y, dA.z, dA.w};
    store_states(parts.A + row * a.states, p.first, a.states, sum);
    if (p.own == 0) parts.skip[row] = own[0], parts.dt_bias[row] = own[1];
    if (g.dfirst) {
      const f32x4 r = late[tiles & 1][i][lane];
      const Four first = {r.x, r.y, r.z, r.w};
      store_states(g.dfirst + row * a.states, p.first, a.states, first);
    }
  }
}

// dB and dC: the sums over `count` blocks of channel groups.
template <typename T>
__global__ __launch_bounds__(256) void ssm_sum_kernel(const float* __restrict__ parts, int64_t count, int64_t rows,
                                                      int wide, int states, void* __restrict__ dB, void* __restrict__ dC) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, size = rows * 2 * wide;
  if (i >= size) return;
  const int n = (int)(i % wide);
  if (n >= states) return;
  float sum = 0.0f;
#pragma unroll 8
  for (int64_t k = 0; k < count; ++k) sum += parts[k * size + i];
  store_one<T>(i / wide % 2 ? dC : dB, i / (2 * wide) * states + n, sum);
}

// dA, dskip and ddt_bias: the sums over the sequences.
__global__ __launch_bounds__(256) void ssm_batch_kernel(const SsmParts parts, int64_t batch, int64_t dim, int states,
                                                        float* __restrict__ dA, float* __restrict__ dskip,
                                                        float* __restrict__ ddt_bias) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = dim * states;
  if (i < n) {
    float sum = 0.0f;
    for (int64_t b = 0; b < batch; ++b) sum += parts.A[b * n + i];
    dA[i] = sum;
  }
  if (i < dim) {
    float s = 0.0f, t = 0.0f;
    for (int64_t b = 0; b < batch; ++b) s += parts.skip[b * dim + i], t += parts.dt_bias[b * dim + i];
    if (dskip) dskip[i] = s;
    if (ddt_bias) ddt_bias[i] = t;
  }
}

int64_t over(int64_t n, int64_t by) { return (n + by - 1) / by; }
int lanes_of(int states) {
  int l = 1;
  while (4 * l < states) l *= 2;
  return l;
}

// f(T{}, lanes) for the activations' dtype and the lanes that a channel's states take.
template <typename F>
int by_form(int dtype, int states, F&& f) {
  auto lanes = [&](auto t) {
    switch (lanes_of(states)) {
      case 1: return f(t, std::integral_constant<int, 1>{});
      case 2: return f(t, std::integral_constant<int, 2>{});
      case 4: return f(t, std::integral_constant<int, 4>{});
      case 8: return f(t, std::integral_constant<int, 8>{});
      default: return f(t, std::integral_constant<int, 16>{});
    }
  };
  switch (dtype) {
    case MORPH_DTYPE_F32: return lanes(F32{});
    case MORPH_DTYPE_F16: return lanes(F16{});
    case MORPH_DTYPE_BF16: return lanes(BF16{});
    default: return MORPH_EDTYPE;
  }
}

// Channel groups of a backward workgroup: as many as leave kBackBlocks workgroups, since each
// workgroup's sums over its channels cross HBM twice.
int groups_per_block(int64_t batch, int64_t dim, int lanes) {
  const int64_t groups = over(dim, 64 / lanes) * batch / kBackBlocks;
  return groups < 1 ? 1 : groups > kMostGroups ? kMostGroups : (int)groups;
}

int check(const morph_ssm* a, int dtype) {
  if (!a || a->batch < 0 || a->steps < 0 || a->dim < 0 || a->reserved != 0) return MORPH_EINVAL;
  if (a->states < 1 || a->states > MORPH_SSM_MAX_STATES) return MORPH_ERANGE;
  if (!known_dtype(dtype)) return MORPH_EDTYPE;
  if (a->batch > 0 && a->dim > 0 && (!a->A || (a->steps > 0 && (!a->x || !a->dt || !a->B || !a->C)))) return MORPH_EINVAL;
  const int64_t most = INT64_MAX >> 12;
  if (a->batch > 0 && a->dim > 0 && (a->dim > most / a->batch || a->steps > most / a->batch / a->dim)) return MORPH_ERANGE;
  return MORPH_OK;
}

size_t part_floats(int64_t batch, int64_t steps, int64_t dim, int states) {
  const int lanes = lanes_of(states);
  const int64_t blocks = over(over(dim, 64 / lanes), groups_per_block(batch, dim, lanes));
  return (size_t)(blocks * batch * steps) * 8 * (size_t)lanes;
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" int morph_ssm_forward(const morph_ssm* a, int dtype, void* y, float* last, float* kept, void* stream) {
  if (const int rc = check(a, dtype)) return rc;
  if (a->batch == 0 || a->dim == 0) return MORPH_OK;
  if ((a->steps > 0 && !y) || !last) return MORPH_EINVAL;
  return by_form(dtype, a->states, [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    if (a->steps == 1) {
      const int64_t groups = over(a->dim, 256 / L);
      if (!launchable(groups * a->batch, 256)) return (int)MORPH_ERANGE;
      hipLaunchKernelGGL((ssm_one_kernel<T, L>), dim3((unsigned)(groups * a->batch)), dim3(256), 0, as_stream(stream), *a,
                         groups, y, last, kept);
      return launch_status();
    }
    const int64_t groups = over(a->dim, 64 / L);
    if (!launchable(groups * a->batch, 64 * kW)) return (int)MORPH_ERANGE;
    hipLaunchKernelGGL((ssm_kernel<T, L>), dim3((unsigned)(groups * a->batch)), dim3(64 * kW), 0, as_stream(stream), *a,
                       groups, y, last, kept);
    return launch_status();
  });
}

extern "C" size_t morph_ssm_workspace_bytes(int64_t batch, int64_t steps, int64_t dim, int states) {
  if (batch < 0 || steps < 0 || dim < 0 || states < 1 || states > MORPH_SSM_MAX_STATES) return 0;
  return (part_floats(batch, steps, dim, states) + (size_t)(batch * dim) * (size_t)(states + 2)) * sizeof(float);
}

extern "C" int morph_ssm_backward(const morph_ssm* a, int dtype, const float* kept, const void* dy, int64_t dy_batch,
                                  int64_t dy_step, const float* dlast, const morph_ssm_grads* g, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (const int rc = check(a, dtype)) return rc;
  if (!g) return MORPH_EINVAL;
  if (a->dim == 0) return MORPH_OK;
  if (!g->dA || (a->skip && !g->dskip) || (a->dt_bias && !g->ddt_bias)) return MORPH_EINVAL;
  if (a->batch > 0 && a->steps > 0 && (!kept || !dy || !g->dx || !g->ddt || !g->dB || !g->dC || (a->z && !g->dz)))
    return MORPH_EINVAL;
  const size_t need = morph_ssm_workspace_bytes(a->batch, a->steps, a->dim, a->states);
  if (need > 0 && (!workspace || workspace_bytes < need)) return MORPH_EWORKSPACE;
  SsmParts parts;
  parts.bc = static_cast<float*>(workspace);
  parts.A = parts.bc + part_floats(a->batch, a->steps, a->dim, a->states);
  parts.skip = parts.A + a->batch * a->dim * a->states;
  parts.dt_bias = parts.skip + a->batch * a->dim;
  hipStream_t s = as_stream(stream);
  const int64_t rows = a->batch * a->steps, sums = over(rows * 8 * lanes_of(a->states), 256);
  const int64_t ends = over(a->dim * a->states, 256);
  if (!launchable(sums, 256) || !launchable(ends, 256)) return MORPH_ERANGE;
  const int rc = by_form(dtype, a->states, [&](auto t, auto lanes) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    if (a->batch == 0) return (int)MORPH_OK;
    const int per = groups_per_block(a->batch, a->dim, L);
    const int64_t blocks = over(over(a->dim, 64 / L), per);
    if (!launchable(blocks * a->batch, 64 * kW)) return (int)MORPH_ERANGE;
    hipLaunchKernelGGL((ssm_back_kernel<T, L>), dim3((unsigned)(blocks * a->batch)), dim3(64 * kW), 0, s, *a, blocks, per,
                       kept, dy, dy_batch, dy_step, dlast, *g, parts);
    if (const int status = launch_status()) return status;
    if (rows == 0) return (int)MORPH_OK;
    hipLaunchKernelGGL(ssm_sum_kernel<T>, dim3((unsigned)sums), dim3(256), 0, s, parts.bc, blocks, rows, 4 * L, a->states,
                       g->dB, g->dC);
    return launch_status();
  });
  if (rc != MORPH_OK) return rc;
  hipLaunchKernelGGL(ssm_batch_kernel, dim3((unsigned)ends), dim3(256), 0, s, parts, a->batch, a->dim, a->states, g->dA,
                     g->dskip, g->ddt_bias);
  return launch_status();
}
