// Selective state space scan (morph_state_space.h) and its backward pass: h_t = exp(d_t A) h_(t-1) + d_t x_t B_t for
// every state of every channel, y = C_t . h_t + skip x, along the steps.
//
// A step costs each state an exponential (which issues for as long as two other instructions) and four to seven more
// instructions, so with 16 states a channel arithmetic bounds the scan, more than twice above what HBM does; the layout
// is for that.  4 x 1024 steps of 5120 channels of 16 states in BF16: forward 160 us, of which vector instructions' issue takes
// 108, backward 383, of which it takes 302, and 20 for the sums.  A lane has four states of a channel, kLanes neighbouring lanes the channel, a wave 64 / kLanes
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
#include <initializer_list>

#include "stage.h"

namespace morph {
namespace {

constexpr int kT = 8;  // steps of a wave
constexpr int kW = 4;  // waves
static_assert(kT * kW == MORPH_SSM_SPAN, "a backward tile begins with a kept state");
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr int kMostGroups = 2;     // channel groups of a backward workgroup
constexpr int kSequences = 4;      // of a lane in a single step: 13.0 us for 64 x 5120 x 16, 13.8 with one, 17.0 with eight
constexpr int kBusy = 512;         // workgroups that keep the chip busy, so that sequences stay whole
constexpr int kFull = 1024;        // workgroups that it holds at a time
constexpr int kBackFull = 768;     // and of the backward
// Tiles of a segment from which 16 waves take its steps in the launch that finds its ends, otherwise 4: 32768 steps of 2048 channels in
// segments of 128 tiles 227 us (4 waves: 257), 3 x 777 of 1100 in segments of 3 tiles 14.3 (13.4).
constexpr int kManyTiles = 16;
constexpr int kJoined = 16;        // segments up to which those that need a segment's first state join it themselves

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
  if constexpr (L == 2) return dpp<K | K << 2 | (2 + K) << 4 | (2 + K) << 6>(x);
  else if constexpr (L == 4) return dpp<K * 0x55>(x);
  else  // lane (l & ~(L - 1)) | K of 32
    return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), (0x1F & ~(L - 1)) | K << 5));
}
// The sum over a channel's lanes, in each.
template <int L>
__device__ __forceinline__ float channel_sum(float x) {
  x += dpp<0xB1>(x);                          // quad_perm [1,0,3,2]
  if constexpr (L >= 4) x += dpp<0x4E>(x);    // quad_perm [2,3,0,1]
  if constexpr (L >= 8) x += dpp<0x141>(x);   // row_half_mirror
  if constexpr (L >= 16) x += dpp<0x140>(x);  // row_mirror
  return x;
}

// The sums over a channel's lanes of kT values, each to the lane whose step it is.  With four lanes a channel four
// steps are summed together: each pair takes one addition and two selections between lanes that differ in
// one bit, and half as many pairs are left for the other.
template <int L>
struct Sums {
  float held[4], out[L <= kT ? kT / L : 1];
  // The value of step t, all of them in descending order.
  template <int t>
  __device__ __forceinline__ void take(float x, int own) {
    if constexpr (L == 4) {
      held[t % 4] = x;
      if constexpr (t % 4 == 0) {
        const bool odd = own & 1, high = own & 2;
        const float a = (odd ? held[1] : held[0]) + dpp<0xB1>(odd ? held[0] : held[1]);  // quad_perm [1,0,3,2]
        const float b = (odd ? held[3] : held[2]) + dpp<0xB1>(odd ? held[2] : held[3]);
        out[t / 4] = (high ? b : a) + dpp<0x4E>(high ? a : b);  // quad_perm [2,3,0,1]
      }
    } else {
      const float s = channel_sum<L>(x);
      if (own == t % L) out[t / L] = s;
    }
  }
};

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

// Four of a step's inputs from `first` on, of n; 0 behind them.
template <typename T>
__device__ __forceinline__ void load_inputs(const char* row, int first, int n, Four& x) {
  if (n % 4 == 0) {
    typedef uint32_t pair __attribute__((ext_vector_type(2), aligned(2)));
    typedef std::conditional_t<std::is_same_v<T, F32>, f32x4_any, pair> four;
    const four v = *reinterpret_cast<const four*>(row + (first < n ? first : 0) * Fmt<T>::bytes);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same_v<T, F32>) x[j] = first < n ? v[j] : 0.0f;
      else x[j] = first < n ? to_float<T>(j % 2 ? v[j / 2] >> 16 : v[j / 2] & 0xFFFFu) : 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = first + j < n ? load_one<T>(row, first + j) : 0.0f;
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
template <typename T>
__device__ __forceinline__ float bits_value(uint32_t w) {
  if constexpr (std::is_same_v<T, F32>) return __builtin_bit_cast(float, w);
  else return to_float<T>(w);
}
// A value of T at a wave-uniform address and a lane's offset in bytes.
template <typename T>
__device__ __forceinline__ uint32_t load_bits(const void* base, uint32_t offset) {
  return *reinterpret_cast<const typename Bits<T>::type*>(static_cast<const char*>(base) + offset);
}
template <typename T>
__device__ __forceinline__ void store_at(void* base, uint32_t offset, float x) {
  char* to = static_cast<char*>(base) + offset;
  if constexpr (std::is_same_v<T, F32>) *reinterpret_cast<float*>(to) = x;
  else *reinterpret_cast<uint16_t*>(to) = (uint16_t)pack2<T>(x, x);
}

// A tensor's rows: where the first step of a sequence begins, and strides in bytes.
struct View {
  const char* at;
  int64_t batch;
  int32_t step;
};

// What the kernels walk.  A sequence is cut into `segments` of `per` tiles each.
struct Scan {
  View x, dt, z, B, C, dy;
  const float* A;
  const float* skip;
  const float* dt_bias;
  int32_t batch, steps, dim, states, tiles, groups, segments, per;
};

// A lane's place: its channel, four of its states and, of a wave's kT steps, those whose per-channel work it does.
// Lanes past the last channel repeat it and store nothing.
template <int L>
struct Lane {
  static constexpr int kR = L <= kT ? kT / L : 1;  // steps of each lane: own + i L
  static constexpr int kC = 64 / L;                // channels of a wave
  int group0, ch, own, first, inside;              // group0: the group's first channel, inside: of the group
  bool active;
  __device__ __forceinline__ Lane(int group, int dim) {
    const int lane = threadIdx.x & 63;
    own = lane % L, first = own * 4;
    group0 = group * kC;
    const int left = dim - group0 < kC ? dim - group0 : kC;
    active = lane / L < left;
    inside = active ? lane / L : left - 1;
    ch = group0 + inside;
  }
  // Whether all lanes have all of their steps, of which `left` are there.
  __device__ __forceinline__ bool whole(int dim, int left) const { return left >= kT && dim - group0 >= kC && L <= kT; }
  __device__ __forceinline__ bool has(int i, int left) const { return active && own + i * L < left && own < kT; }
};

// A wave's kT steps from t0 on; in place of those behind the sequence's last, that one.  (Loads under a condition
// would be waited for where its branches meet, and so would those of one tensor before the condition for the next: a
// kernel that loads ahead finds all of its offsets first, then loads.  4 x 1024 steps of 2560 channels of 16 states in
// BF16, forward: 78 us, tensor by tensor 83.)
struct Span {
  int t0, left;
  __device__ __forceinline__ Span(int t, int steps) : t0(t < steps ? t : steps - 1), left(steps - t0) {}
  __device__ __forceinline__ bool whole() const { return left >= kT; }
  // The first step's row of a sequence, a wave-uniform address.
  __device__ __forceinline__ const char* row(const View& v, int b) const { return v.at + b * v.batch + (int64_t)t0 * v.step; }
};

// A channel and step tensor's values of a wave's steps.
template <typename T, int L>
struct Rows {
  uint32_t w[Lane<L>::kR], at[Lane<L>::kR];
  // The lane's first step's offset in bytes; its others' are added to the address.
  static __device__ __forceinline__ uint32_t offset(const Lane<L>& p, int step) {
    return (uint32_t)(p.own < kT ? p.own : kT - 1) * (uint32_t)step + (uint32_t)p.inside * Fmt<T>::bytes;
  }
  __device__ __forceinline__ void place_whole(const Lane<L>& p, const View& v) {
#pragma unroll
    for (int i = 0; i < Lane<L>::kR; ++i) at[i] = offset(p, v.step);
  }
  __device__ __forceinline__ void place_part(const Lane<L>& p, const View& v, const Span& s) {
#pragma unroll
    for (int i = 0; i < Lane<L>::kR; ++i) {
      const int t = p.own + i * L;
      at[i] = (uint32_t)(t < s.left ? t : s.left - 1) * (uint32_t)v.step + (uint32_t)p.inside * Fmt<T>::bytes;
    }
  }
  __device__ __forceinline__ void load(const Lane<L>& p, const View& v, int b, const Span& s) {
    const char* row = s.row(v, b) + p.group0 * Fmt<T>::bytes;
    const int64_t next = s.whole() ? (int64_t)L * v.step : 0;
#pragma unroll
    for (int i = 0; i < Lane<L>::kR; ++i) w[i] = load_bits<T>(row + i * next, at[i]);
  }
  // Both, where nothing is computed between loads and use: with all offsets in vector registers.
  __device__ __forceinline__ void fetch(const Lane<L>& p, const View& v, int b, const Span& s) {
    const char* row = s.row(v, b) + p.group0 * Fmt<T>::bytes;
    if (s.whole()) {
#pragma unroll
      for (int i = 0; i < Lane<L>::kR; ++i) at[i] = offset(p, v.step) + (uint32_t)(i * L) * (uint32_t)v.step;
    } else {
      place_part(p, v, s);
    }
#pragma unroll
    for (int i = 0; i < Lane<L>::kR; ++i) w[i] = load_bits<T>(row, at[i]);
  }
  __device__ __forceinline__ float operator[](int i) const { return bits_value<T>(w[i]); }
};

// B or C of a wave's steps on its way from memory to the wave's part of LDS, [kT][4 L] floats; 0 for states
// and steps that are not there.
template <typename T, int L>
struct Inputs {
  static constexpr int kCount = L / 2;
  uint32_t w[kCount], at[kCount];
  static __device__ __forceinline__ int step_of(int i) { return (i * 64 + (int)(threadIdx.x & 63)) / (4 * L); }
  static __device__ __forceinline__ int state_of(int i) { return (i * 64 + (int)(threadIdx.x & 63)) % (4 * L); }
  static __device__ __forceinline__ uint32_t offset(int i, int t, int step, int states) {
    const int n = state_of(i);
    return (uint32_t)t * (uint32_t)step + (uint32_t)(n < states ? n : states - 1) * Fmt<T>::bytes;
  }
  __device__ __forceinline__ void place_whole(const View& v, int states) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) at[i] = offset(i, step_of(i), v.step, states);
  }
  __device__ __forceinline__ void place_part(const View& v, const Span& s, int states) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int t = step_of(i);
      at[i] = offset(i, t < s.left ? t : s.left - 1, v.step, states);
    }
  }
  __device__ __forceinline__ void load(const View& v, int b, const Span& s) {
    const char* row = s.row(v, b);
#pragma unroll
    for (int i = 0; i < kCount; ++i) w[i] = load_bits<T>(row, at[i]);
  }
  __device__ __forceinline__ void fetch(const View& v, int b, const Span& s, int states) {
    const char* row = s.row(v, b);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      int t = step_of(i);
      if (!s.whole()) t = t < s.left ? t : s.left - 1;
      at[i] = offset(i, t, v.step, states);
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) w[i] = load_bits<T>(row, at[i]);
  }
  // (What is not there is told apart here: looked at in load, the loads would be waited for there.)
  __device__ __forceinline__ void put(float* to, int left, int states) const {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int v = i * 64 + (threadIdx.x & 63);
      const bool there = state_of(i) < states && step_of(i) < left;
      to[v] = there ? bits_value<T>(w[i]) : 0.0f;
    }
  }
};

// The states of a channel in a tensor [.., dim, states], `row` its sequence.
__device__ __forceinline__ int64_t states_at(const Scan& a, int64_t row, int ch) { return (row * a.dim + ch) * a.states; }

// What enters a segment, four states of a channel: behind few segments joined here, from `start` on through one after the
// other, what more than kJoined leave is there (ssm_join_kernel).  kBack: from the last segment on.
template <bool kBack>
__device__ __forceinline__ void entering_states(const Scan& a, int segment, int b, int ch, int first, const Four& A2,
                                                const float* start, const float* ends, const float* sums, Four& s) {
  const int last = kBack ? a.segments - 1 : 0;
  if (segment != last && a.segments > kJoined) {
    load_states(ends + states_at(a, (int64_t)segment * a.batch + b, ch), first, a.states, s);
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s[j] = 0.0f;
  if (start) load_states(start + states_at(a, b, ch), first, a.states, s);
  for (int k = last; k != segment;) {
    k += kBack ? -1 : 1;
    const int64_t row = (int64_t)k * a.batch + b;
    Four S;
    load_states(ends + states_at(a, row, ch), first, a.states, S);
    const float d = sums[row * a.dim + ch];
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] = __fmaf_rn(__builtin_amdgcn_exp2f(d * A2[j]), s[j], S[j]);
  }
}

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

// What a lane needs of its channel throughout.
struct Channel {
  Four A2;  // A log2(e)
  float skip, bias;
};
template <int L>
__device__ __forceinline__ Channel load_channel(const Scan& a, const Lane<L>& p) {
  Channel c;
  load_states(a.A + (int64_t)p.ch * a.states, p.first, a.states, c.A2);
  c.skip = a.skip ? a.skip[p.ch] : 0.0f;
  c.bias = a.dt_bias ? a.dt_bias[p.ch] : 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) c.A2[j] *= kLog2e;
  return c;
}

template <typename T, int L, bool kGated>
__global__ __launch_bounds__(64 * kW, L < 4 ? 3 : 4) void ssm_kernel(const Scan a, const float* __restrict__ first,
                                                                        const float* __restrict__ from,
                                                                        const float* __restrict__ sums,
                                                                        char* __restrict__ y, float* __restrict__ last,
                                                                        float* __restrict__ kept) {
  constexpr int kR = Lane<L>::kR;
  __shared__ float bc[kW][2][kT * 4 * L];
  __shared__ f32x4 ends[2][kW][2][64];
  const int group = (int)blockIdx.x % a.groups, rest = (int)blockIdx.x / a.groups;
  const int segment = rest % a.segments, b = rest / a.segments;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const Lane<L> p(group, a.dim);
  const Channel c = load_channel(a, p);
  Four carry;
  entering_states<false>(a, segment, b, p.ch, p.first, c.A2, first, from, sums, carry);
  const int begin = segment * a.per, end = begin + a.per < a.tiles ? begin + a.per : a.tiles;

  Rows<T, L> rx, rd, rz;
  Inputs<T, L> inB, inC;
  auto fetch = [&](int tile) {
    const Span s((tile * kW + wave) * kT, a.steps);
    if constexpr (L > 4) {  // the registers that all offsets take are not there: 64 states 234 us, with them 244 to 252
      rx.fetch(p, a.x, b, s), rd.fetch(p, a.dt, b, s);
      if constexpr (kGated) rz.fetch(p, a.z, b, s);
      inB.fetch(a.B, b, s, a.states), inC.fetch(a.C, b, s, a.states);
      return;
    }
    rx.place_whole(p, a.x), rd.place_whole(p, a.dt);
    if constexpr (kGated) rz.place_whole(p, a.z);
    inB.place_whole(a.B, a.states), inC.place_whole(a.C, a.states);
    if (!s.whole()) {
      rx.place_part(p, a.x, s), rd.place_part(p, a.dt, s);
      if constexpr (kGated) rz.place_part(p, a.z, s);
      inB.place_part(a.B, s, a.states), inC.place_part(a.C, s, a.states);
    }
    rx.load(p, a.x, b, s), rd.load(p, a.dt, b, s);
    if constexpr (kGated) rz.load(p, a.z, b, s);
    inB.load(a.B, b, s), inC.load(a.C, b, s);
  };
  if (begin < end) fetch(begin);
  for (int tile = begin; tile < end; ++tile) {
    const int t0 = (tile * kW + wave) * kT, left = a.steps - t0;
    const bool whole = p.whole(a.dim, left);
    float x[kR], d[kR], u[kR], z[kR];
    float* B = bc[wave][0];
    float* C = bc[wave][1];
    inB.put(B, left, a.states), inC.put(C, left, a.states);
    wave_order();
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      x[i] = rx[i];
      if constexpr (kGated) z[i] = rz[i];
      d[i] = softplus(rd[i] + c.bias);
      if (!whole && !p.has(i, left)) d[i] = x[i] = 0.0f;
      u[i] = d[i] * x[i];
    }
    if (tile + 1 < end) fetch(tile + 1);
    if (kept && wave == 0 && p.active)
      store_states(kept + states_at(a, (int64_t)b * a.tiles + tile, p.ch), p.first, a.states, carry);
    Four P[kT], h[kT];
    walk<L, true>(d, u, c.A2, B, p.first, P, h);
    const int turn = tile & 1;  // every wave has passed the barrier behind the last use of this half
    ends[turn][wave][0][lane] = as_vector(P[kT - 1]);
    ends[turn][wave][1][lane] = as_vector(h[kT - 1]);
    __syncthreads();
    Four enter;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      if (w == wave) {
#pragma unroll
        for (int j = 0; j < 4; ++j) enter[j] = carry[j];
      }
      const f32x4 A = ends[turn][w][0][lane], S = ends[turn][w][1][lane];
#pragma unroll
      for (int j = 0; j < 4; ++j) carry[j] = __fmaf_rn(A[j], carry[j], S[j]);
    }
    Sums<L> sums = {};
    each_step<kT>([&](auto step) {
      constexpr int t = kT - 1 - decltype(step)::value;
      const f32x4 ct = *reinterpret_cast<const f32x4*>(C + t * 4 * L + p.first);
      float s = ct[0] * __fmaf_rn(P[t][0], enter[0], h[t][0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) s = __fmaf_rn(ct[j], __fmaf_rn(P[t][j], enter[j], h[t][j]), s);
      sums.template take<t>(s, p.own);
    });
    wave_order();
    if (left <= 0) continue;
    char* rows = y + (((int64_t)b * a.steps + t0) * a.dim + p.group0) * Fmt<T>::bytes;
    const uint32_t to = Rows<T, L>::offset(p, a.dim * Fmt<T>::bytes);
#pragma unroll
    for (int i = 0; i < kR; ++i) {
      float s = __fmaf_rn(c.skip, x[i], sums.out[i]);
      if constexpr (kGated) s *= z[i] * gate_sigmoid(z[i]);
      if (whole || p.has(i, left)) store_at<T>(rows + (int64_t)(i * L) * a.dim * Fmt<T>::bytes, to, s);
    }
  }
  if (segment == a.segments - 1 && wave == 0 && p.active)
    store_states(last + states_at(a, b, p.ch), p.first, a.states, carry);
}

// What a segment does to a state that passes through it, for the segments to be walked side by side: the product of its
// gates is exp(A times the sum of d), and `ends` its result from a zero state (kBack: of the gradients r, from its last
// step to its first).  Each wave takes its part of the segment's steps; no output, so neither skip nor dB and dC.
// segment s: ends[s + 1], sums[s + 1] (kBack: s - 1), where what enters the next one then is joined.
template <typename T, int L, bool kBack, bool kGated, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void ssm_ends_kernel(const Scan a, float* __restrict__ ends, float* __restrict__ sums) {
  constexpr int kR = Lane<L>::kR;
  __shared__ float bc[kWaves][kT * 4 * L];
  __shared__ f32x4 join[kWaves][2][64];
  __shared__ float whole_sum[kWaves][64];
  const int group = (int)blockIdx.x % a.groups, rest = (int)blockIdx.x / a.groups;
  const int segment = rest % (a.segments - 1) + (kBack ? 1 : 0), b = rest / (a.segments - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const Lane<L> p(group, a.dim);
  const Channel c = load_channel(a, p);
  // runs of kT steps: all of the segment's, and from the wave's first on (kBack: its last, downwards) how many it takes
  const int all = a.per * kW, each = (all + kWaves - 1) / kWaves, before = wave * each;
  const int count = before >= all ? 0 : all - before < each ? all - before : each;
  const int run0 = segment * all + (kBack ? before + count - 1 : before);
  Rows<T, L> rd, rx, rz;  // x: kBack: dy
  Inputs<T, L> in;
  float* mine = bc[wave];
  float sum = 0.0f;
  Four s = {};
  auto fetch = [&](int i) {
    const Span s((run0 + (kBack ? -i : i)) * kT, a.steps);
    const View &x = kBack ? a.dy : a.x, &v = kBack ? a.C : a.B;
    rd.place_whole(p, a.dt), rx.place_whole(p, x);
    if constexpr (kGated) rz.place_whole(p, a.z);
    in.place_whole(v, a.states);
    if (!s.whole()) {
      rd.place_part(p, a.dt, s), rx.place_part(p, x, s);
      if constexpr (kGated) rz.place_part(p, a.z, s);
      in.place_part(v, s, a.states);
    }
    rd.load(p, a.dt, b, s), rx.load(p, x, b, s);
    if constexpr (kGated) rz.load(p, a.z, b, s);
    in.load(v, b, s);
  };
  if (count > 0) fetch(0);
  for (int i = 0; i < count; ++i) {
    const int t0 = (run0 + (kBack ? -i : i)) * kT, left = a.steps - t0;
    const bool whole = p.whole(a.dim, left);
    float d[kR], u[kR];
    in.put(mine, left, a.states);
    wave_order();
#pragma unroll
    for (int k = 0; k < kR; ++k) {
      d[k] = softplus(rd[k] + c.bias);
      u[k] = rx[k];
      if constexpr (kBack) {
        if constexpr (kGated) u[k] *= silu(rz[k]).y;
      } else {
        u[k] *= d[k];
      }
      if (!whole && !p.has(k, left)) d[k] = u[k] = 0.0f;
      sum += d[k];
    }
    if (i + 1 < count) fetch(i + 1);
    each_step<kT>([&](auto step) {
      constexpr int t = kBack ? kT - 1 - decltype(step)::value : decltype(step)::value;
      const float dt = spread<L, t % L>(d[t / L]), ut = spread<L, t % L>(u[t / L]);
      const f32x4 in_t = *reinterpret_cast<const f32x4*>(mine + t * 4 * L + p.first);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float gate = __builtin_amdgcn_exp2f(dt * c.A2[j]);
        s[j] = kBack ? gate * __fmaf_rn(in_t[j], ut, s[j]) : __fmaf_rn(gate, s[j], in_t[j] * ut);
      }
    });
    wave_order();
  }
  sum = channel_sum<L>(sum);
  Four P;
#pragma unroll
  for (int j = 0; j < 4; ++j) P[j] = __builtin_amdgcn_exp2f(sum * c.A2[j]);
  join[wave][0][lane] = as_vector(P), join[wave][1][lane] = as_vector(s);
  whole_sum[wave][lane] = sum;
  __syncthreads();
  if (wave != 0) return;
  Four out = {};
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const int w = kBack ? kWaves - 1 - i : i;
    const f32x4 A = join[w][0][lane], S = join[w][1][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = __fmaf_rn(A[j], out[j], S[j]);
    sum += whole_sum[w][lane];
  }
  if (!p.active) return;
  const int64_t row = (int64_t)(segment + (kBack ? -1 : 1)) * a.batch + b;
  store_states(ends + states_at(a, row, p.ch), p.first, a.states, out);
  if (p.own == 0) sums[row * a.dim + p.ch] = sum;
}

// What enters each segment, in place of `ends`: from `first` through one after the other (kBack: from the last, NULL: zeros).
template <bool kBack>
__global__ __launch_bounds__(256) void ssm_join_kernel(const Scan a, const float* __restrict__ first, float* __restrict__ ends,
                                                       const float* __restrict__ sums) {
  const int64_t size = (int64_t)a.batch * a.dim * a.states, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= size) return;
  const float A2 = a.A[i % ((int64_t)a.dim * a.states)] * kLog2e;
  float s = first ? first[i] : 0.0f;
  for (int k = 1; k < a.segments; ++k) {
    const int64_t row = kBack ? a.segments - 1 - k : k;
    s = __fmaf_rn(__builtin_amdgcn_exp2f(sums[row * a.batch * a.dim + i / a.states] * A2), s, ends[row * size + i]);
    ends[row * size + i] = s;
  }
}

// One step: the state crosses once in and once out, and HBM bounds it.  A lane takes its states of kSequences sequences, whose
// loads are all issued first.
template <typename T, int L>
__global__ __launch_bounds__(256) void ssm_one_kernel(const Scan a, int groups, const float* __restrict__ first_state,
                                                      char* __restrict__ y, float* __restrict__ last,
                                                      float* __restrict__ kept) {
  const int lane = threadIdx.x, own = lane % L, first = own * 4;
  const int ch = ((int)blockIdx.x % groups) * (256 / L) + lane / L, b0 = ((int)blockIdx.x / groups) * kSequences;
  if (ch >= a.dim) return;  // whole channels: their lanes are together
  Four A, h[kSequences], B[kSequences], C[kSequences];
  float x[kSequences], z[kSequences], d[kSequences];
#pragma unroll
  for (int i = 0; i < kSequences; ++i) {
    const int b = b0 + i < a.batch ? b0 + i : a.batch - 1;
    if (first_state) {
      load_states(first_state + states_at(a, b, ch), first, a.states, h[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) h[i][j] = 0.0f;
    }
    load_inputs<T>(a.B.at + b * a.B.batch, first, a.states, B[i]);
    load_inputs<T>(a.C.at + b * a.C.batch, first, a.states, C[i]);
    x[i] = load_one<T>(a.x.at + b * a.x.batch, ch), d[i] = load_one<T>(a.dt.at + b * a.dt.batch, ch);
    z[i] = a.z.at ? load_one<T>(a.z.at + b * a.z.batch, ch) : 0.0f;
  }
  load_states(a.A + (int64_t)ch * a.states, first, a.states, A);
  const float bias = a.dt_bias ? a.dt_bias[ch] : 0.0f, skip = a.skip ? a.skip[ch] : 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) A[j] *= kLog2e;
#pragma unroll
  for (int i = 0; i < kSequences; ++i) {
    if (b0 + i >= a.batch) break;
    const int64_t at = states_at(a, b0 + i, ch);
    if (kept) store_states(kept + at, first, a.states, h[i]);
    const float step = softplus(d[i] + bias), u = step * x[i];
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[i][j] = __fmaf_rn(__builtin_amdgcn_exp2f(step * A[j]), h[i][j], u * B[i][j]);
      s = __fmaf_rn(C[i][j], h[i][j], s);
    }
    store_states(last + at, first, a.states, h[i]);
    s = __fmaf_rn(skip, x[i], channel_sum<L>(s));
    if (a.z.at) s *= z[i] * gate_sigmoid(z[i]);
    if (own == 0) store_one<T>(y, (int64_t)(b0 + i) * a.dim + ch, s);
  }
}

// Where a backward's sums lie in its workspace.
struct SsmParts {
  float* bc;       // [blocks of channel groups][batch][steps][2][4 L]: dB, dC
  float* A;        // [segments][batch][dim][states]
  float* skip;     // [segments][batch][dim]
  float* dt_bias;  // [segments][batch][dim]
  float* late;     // [segments][batch][dim][states]: r behind each segment, times its gate
  float* sums;     // [segments][batch][dim]
};

// A sequence's channel groups go to `blocks` workgroups, to the first ones one more where they do not come out even.
template <typename T, int L, bool kGated>
__global__ __launch_bounds__(64 * kW, L < 16 ? 3 : 2) void ssm_back_kernel(const Scan a, int blocks,
                                                                           const float* __restrict__ kept,
                                                                           const float* __restrict__ dlast,
                                                                           const morph_ssm_grads g, const SsmParts parts) {
  constexpr int kR = Lane<L>::kR, kRep = 16 / L, kSlots = kRep < kT ? kT / kRep : 1;
  __shared__ float bc[kW][2][kT * 4 * L];
  __shared__ f32x4 ends[2][kW][3][64];
  __shared__ f32x4 late[2][kMostGroups][64];           // r behind the tile, times its gate
  __shared__ f32x4 sum_A[kMostGroups][kW][64];         // dA of each wave's steps
  __shared__ float sum_own[kMostGroups][kW][2][64];    // dskip, ddt_bias
  // the larger workgroups of all sequences first
  const int rows = a.segments * a.batch, block = (int)blockIdx.x / rows, rest = (int)blockIdx.x % rows;
  const int segment = rest % a.segments, b = rest / a.segments;
  const int per = a.groups / blocks, more = a.groups % blocks;
  const int group0 = block * per + (block < more ? block : more), count = per + (block < more ? 1 : 0);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int begin = segment * a.per, end = begin + a.per < a.tiles ? begin + a.per : a.tiles;
  for (int i = 0; i < count; ++i) {
    const Lane<L> p(group0 + i, a.dim);
    sum_A[i][wave][lane] = f32x4{0, 0, 0, 0};
    sum_own[i][wave][0][lane] = sum_own[i][wave][1][lane] = 0.0f;
    if (wave == 0) {
      Four r;
      entering_states<true>(a, segment, b, p.ch, p.first, load_channel(a, p).A2, dlast, parts.late, parts.sums, r);
      late[0][i][lane] = as_vector(r);
    }
  }
  Inputs<T, L> inB, inC;
  float* B = bc[wave][0];
  float* C = bc[wave][1];
  int half = 0, turn = 0;
  for (int tile = end - 1; tile >= begin; --tile, turn ^= 1) {
    const int t0 = (tile * kW + wave) * kT, left = a.steps - t0;
    const Span span(t0, a.steps);
    inB.fetch(a.B, b, span, a.states), inC.fetch(a.C, b, span, a.states);
    inB.put(B, left, a.states), inC.put(C, left, a.states);
    wave_order();
    float acc[kSlots][2] = {};
    for (int i = 0; i < count; ++i, half ^= 1) {
      const Lane<L> p(group0 + i, a.dim);
      const bool whole = p.whole(a.dim, left);
      Rows<T, L> rx, rd, rz, re;
      rx.fetch(p, a.x, b, span), rd.fetch(p, a.dt, b, span), re.fetch(p, a.dy, b, span);
      if constexpr (kGated) rz.fetch(p, a.z, b, span);
      const Channel c = load_channel(a, p);
      Four enter;
      load_states(kept + states_at(a, (int64_t)b * a.tiles + tile, p.ch), p.first, a.states, enter);
      float x[kR], d[kR], u[kR], raw[kR], ds[kR], slope[kR];  // slope: of silu(z), times dy
#pragma unroll
      for (int k = 0; k < kR; ++k) {
        x[k] = rx[k], raw[k] = rd[k] + c.bias, ds[k] = re[k];
        d[k] = softplus(raw[k]);
        if constexpr (kGated) {
          const Silu q = silu(rz[k]);
          slope[k] = ds[k] * q.slope, ds[k] *= q.y;
        }
        if (!whole && !p.has(k, left)) d[k] = x[k] = ds[k] = 0.0f;
        u[k] = d[k] * x[k];
      }
      Four gate[kT], h[kT];
      walk<L, false>(d, u, c.A2, B, p.first, gate, h);
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
        const f32x4 ct = *reinterpret_cast<const f32x4*>(C + t * 4 * L + p.first);
#pragma unroll
        for (int j = 0; j < 4; ++j) Q[j] = gate[t][j] * __fmaf_rn(ct[j], dst, Q[j]);
      });
      ends[half][wave][0][lane] = as_vector(P);
      ends[half][wave][1][lane] = as_vector(h[kT - 1]);
      ends[half][wave][2][lane] = as_vector(Q);
      __syncthreads();  // every wave has passed it behind its last use of this half
      for (int w = 0; w < wave; ++w) {
        const f32x4 Pw = ends[half][w][0][lane], S = ends[half][w][1][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) enter[j] = __fmaf_rn(Pw[j], enter[j], S[j]);
      }
      const f32x4 after = late[turn][i][lane];
      Four r = {after.x, after.y, after.z, after.w};
      for (int w = kW - 1; w > wave; --w) {
        const f32x4 Pw = ends[half][w][0][lane], Qw = ends[half][w][2][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __fmaf_rn(Pw[j], r[j], Qw[j]);
      }
      // the states again, from the true one
      each_step<kT>([&](auto step) {
        constexpr int t = decltype(step)::value;
        const float ut = spread<L, t % L>(u[t / L]);
        const f32x4 Bt = *reinterpret_cast<const f32x4*>(B + t * 4 * L + p.first);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[t][j] = __fmaf_rn(gate[t][j], t ? h[t ? t - 1 : 0][j] : enter[j], ut * Bt[j]);
      });
      Sums<L> rB = {}, wA = {}, Ch = {};
      float pair[4][2];
      const f32x4 before = sum_A[i][wave][lane];
      Four dA = {before.x, before.y, before.z, before.w};
      each_step<kT>([&](auto step) {
        constexpr int t = kT - 1 - decltype(step)::value;
        const float dst = spread<L, t % L>(ds[t / L]), dt = spread<L, t % L>(d[t / L]), ut = spread<L, t % L>(u[t / L]);
        const f32x4 Bt = *reinterpret_cast<const f32x4*>(B + t * 4 * L + p.first);
        const f32x4 ct = *reinterpret_cast<const f32x4*>(C + t * 4 * L + p.first);
        float v[8], sB = 0.0f, sA = 0.0f, sC = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float q = __fmaf_rn(ct[j], dst, r[j]);
          sB = j ? __fmaf_rn(q, Bt[j], sB) : q * Bt[j];
          if constexpr (kGated) sC = j ? __fmaf_rn(ct[j], h[t][j], sC) : ct[j] * h[t][j];
          v[j] = q * ut;
          v[4 + j] = h[t][j] * dst;
          r[j] = gate[t][j] * q;
          const float w = r[j] * (t ? h[t ? t - 1 : 0][j] : enter[j]);
          sA = j ? __fmaf_rn(w, c.A2[j], sA) : w * c.A2[j];
          dA[j] = __fmaf_rn(w, dt, dA[j]);
        }
        rB.template take<t>(sB, p.own);
        wA.template take<t>(sA, p.own);
        if constexpr (kGated) Ch.template take<t>(sC, p.own);
        // over the wave's channels: dB to the lower 32 lanes, dC to the upper; states 0 and 1 to even rows of 16
        // lanes, 2 and 3 to odd ones; then within the rows, with L = 4 four steps together
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          swap32(v[j], v[4 + j]);
          v[j] += v[4 + j];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          swap16(v[j], v[2 + j]);
          v[j] += v[2 + j];
          if constexpr (L == 4) {
            pair[t % 4][j] = v[j];
          } else {
            if constexpr (L <= 8) v[j] += dpp<kRotate8>(v[j]);
            if constexpr (L <= 2) v[j] += dpp<kRotate4>(v[j]);
            if constexpr (L <= 2) v[j] += dpp<kRotate2>(v[j]);
            acc[t / kRep][j] += (lane & 15) / L == t % kRep ? v[j] : 0.0f;
          }
        }
        if constexpr (L == 4 && t % 4 == 0) {
          const bool odd = lane & 4, high = lane & 8;  // step t + (lane >> 2) % 4 stays
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = (high ? pair[2][j] : pair[0][j]) + dpp<kRotate8>(high ? pair[0][j] : pair[2][j]);
            const float y = (high ? pair[3][j] : pair[1][j]) + dpp<kRotate8>(high ? pair[1][j] : pair[3][j]);
            // from 4 lanes before, or for the even ones behind; both by all lanes, since a lane reads active ones only
            const float give = odd ? x : y, before4 = dpp<kRotate4>(give), behind4 = dpp<kRotate12>(give);
            acc[t / 4][j] += (odd ? y : x) + (odd ? before4 : behind4);
          }
        }
        __builtin_amdgcn_sched_barrier(0);  // steps mixed by the scheduler take more registers than there are
      });
      sum_A[i][wave][lane] = as_vector(dA);
      if (wave == 0) late[turn ^ 1][i][lane] = as_vector(r);
      if (left <= 0) continue;
      float dskip = 0.0f, dbias = 0.0f;
      const uint32_t to = Rows<T, L>::offset(p, a.dim * Fmt<T>::bytes);
      const int64_t at = (((int64_t)b * a.steps + t0) * a.dim + p.group0) * Fmt<T>::bytes;
#pragma unroll
      for (int k = 0; k < kR; ++k) {
        const int64_t row = at + (int64_t)(k * L) * a.dim * Fmt<T>::bytes;
        float ddt = __fmaf_rn(x[k], rB.out[k], wA.out[k] * kLn2) * sigmoid(raw[k]).a;
        if (whole || p.has(k, left)) {
          store_at<T>(static_cast<char*>(g.dx) + row, to, __fmaf_rn(d[k], rB.out[k], c.skip * ds[k]));
          store_at<T>(static_cast<char*>(g.ddt) + row, to, ddt);
          if constexpr (kGated) store_at<T>(static_cast<char*>(g.dz) + row, to, __fmaf_rn(c.skip, x[k], Ch.out[k]) * slope[k]);
        } else {
          ddt = 0.0f;
        }
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
      if (t < kT && t < left) {
        float* to = parts.bc + ((((int64_t)block * a.batch + b) * a.steps + t0 + t) * 2 + (lane >> 5)) * 4 * L +
                    (lane & (L - 1)) * 4 + ((lane >> 4) & 1) * 2;
        *reinterpret_cast<f32x2*>(to) = f32x2{acc[s][0], acc[s][1]};
      }
    }
  }
  __syncthreads();
  for (int i = wave; i < count; i += kW) {  // a wave a channel group
    const Lane<L> p(group0 + i, a.dim);
    f32x4 dA = sum_A[i][0][lane];
    float own[2] = {sum_own[i][0][0][lane], sum_own[i][0][1][lane]};
#pragma unroll
    for (int w = 1; w < kW; ++w) {
      dA += sum_A[i][w][lane];
      own[0] += sum_own[i][w][0][lane], own[1] += sum_own[i][w][1][lane];
    }
    own[0] = channel_sum<L>(own[0]), own[1] = channel_sum<L>(own[1]);
    if (!p.active) continue;
    const int64_t row = (int64_t)segment * a.batch + b;
    const Four sum = {dA.x, dA.y, dA.z, dA.w};
    store_states(parts.A + states_at(a, row, p.ch), p.first, a.states, sum);
    if (p.own == 0) parts.skip[row * a.dim + p.ch] = own[0], parts.dt_bias[row * a.dim + p.ch] = own[1];
    if (segment == 0 && g.dfirst) {
      const f32x4 r = late[turn][i][lane];
      const Four first = {r.x, r.y, r.z, r.w};
      store_states(g.dfirst + states_at(a, b, p.ch), p.first, a.states, first);
    }
  }
}

// dB and dC, the sums over `count` blocks of channel groups, by the first workgroups; dA, dskip and ddt_bias, the sums
// over the sequences and their segments, by the others, from workgroup `ends` on.
template <typename T>
__global__ __launch_bounds__(256) void ssm_sum_kernel(const SsmParts parts, int64_t count, int64_t rows, int wide,
                                                      int64_t sequences, int64_t dim, int states, int ends,
                                                      const morph_ssm_grads g) {
  if ((int)blockIdx.x < ends) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, size = rows * 2 * wide;
    if (i >= size) return;
    const int n = (int)(i % wide);
    if (n >= states) return;
    float sum = 0.0f;
#pragma unroll 8
    for (int64_t k = 0; k < count; ++k) sum += parts.bc[k * size + i];
    store_one<T>(i / wide % 2 ? g.dC : g.dB, i / (2 * wide) * states + n, sum);
    return;
  }
  const int64_t i = (int64_t)((int)blockIdx.x - ends) * 256 + threadIdx.x, n = dim * states;
  if (i < n) {
    float sum = 0.0f;
#pragma unroll 4
    for (int64_t b = 0; b < sequences; ++b) sum += parts.A[b * n + i];
    g.dA[i] = sum;
  }
  if (i < dim) {
    float s = 0.0f, t = 0.0f;
#pragma unroll 4
    for (int64_t b = 0; b < sequences; ++b) s += parts.skip[b * dim + i], t += parts.dt_bias[b * dim + i];
    if (g.dskip) g.dskip[i] = s;
    if (g.ddt_bias) g.ddt_bias[i] = t;
  }
}

int64_t over(int64_t n, int64_t by) { return (n + by - 1) / by; }
// Of a channel, four states each; two at least: 4 states take 170 us backward (4 x 1024 steps of 2560 channels in BF16) with two
// lanes, one of them idle, and 287 with one, whose steps' own values do not fit its registers; forward 70 and 67.
int lanes_of(int states) {
  int l = 2;
  while (4 * l < states) l *= 2;
  return l;
}

// f(T{}, lanes, gated) for the activations' dtype and the lanes that a channel's states take.
template <typename F>
int by_form(int dtype, int states, bool gated, F&& f) {
  auto gate = [&](auto t, auto lanes) { return gated ? f(t, lanes, std::true_type{}) : f(t, lanes, std::false_type{}); };
  auto lanes = [&](auto t) {
    switch (lanes_of(states)) {
      case 2: return gate(t, std::integral_constant<int, 2>{});
      case 4: return gate(t, std::integral_constant<int, 4>{});
      case 8: return gate(t, std::integral_constant<int, 8>{});
      default: return gate(t, std::integral_constant<int, 16>{});
    }
  };
  switch (dtype) {
    case MORPH_DTYPE_F32: return lanes(F32{});
    case MORPH_DTYPE_F16: return lanes(F16{});
    case MORPH_DTYPE_BF16: return lanes(BF16{});
    default: return MORPH_EDTYPE;
  }
}

int64_t tiles_of(int64_t steps) { return over(steps, kT * kW); }

// Tiles of a segment.  A scan whose channel groups leave CUs idle is cut into segments that are walked side by side,
// after a launch that finds what each does to a state: two thirds of the scan's own arithmetic, so not where there
// are kBusy workgroups without it.
int64_t tiles_per_segment(int64_t batch, int64_t steps, int64_t groups) {
  const int64_t tiles = tiles_of(steps), blocks = groups * batch;
  if (tiles < 2 || blocks >= kBusy) return tiles > 0 ? tiles : 1;
  int64_t segments = kFull / (blocks > 0 ? blocks : 1);
  if (segments > tiles) segments = tiles;
  return over(tiles, segments);
}

// Workgroups of a backward per sequence and segment: as many as the chip holds at a time, and a channel group for
// each of them at least and kMostGroups at most.  (Each workgroup's sums over its channels cross HBM twice.)
int64_t back_blocks(int64_t batch, int64_t segments, int64_t groups) {
  int64_t n = kBackFull / (batch * segments > 0 ? batch * segments : 1);
  if (n * kMostGroups < groups) n = over(groups, kMostGroups);
  return n < 1 ? 1 : n > groups ? groups : n;
}

// A call's sizes, within what the kernels count in 32 bits, and where its workspace's parts lie.
struct Plan {
  int64_t groups, tiles, per, segments, blocks;
  size_t bc, states, channels;  // floats: dB and dC; a state tensor of all segments; a channel tensor
  Plan(int64_t batch, int64_t steps, int64_t dim, int n) {
    const int lanes = lanes_of(n);
    groups = over(dim, 64 / lanes), tiles = tiles_of(steps), per = tiles_per_segment(batch, steps, groups);
    segments = tiles > 0 ? over(tiles, per) : 1;
    blocks = back_blocks(batch, segments, groups);
    bc = (size_t)(blocks * batch * steps) * 8 * (size_t)lanes;
    channels = (size_t)(segments * batch * dim), states = channels * (size_t)n;
  }
  size_t bytes(bool backward) const {
    const size_t joined = segments > 1 ? states + channels : 0;
    return (backward ? bc + states + 2 * channels + joined : joined) * sizeof(float);
  }
};

int check(const morph_ssm* a, int dtype) {
  if (!a || a->batch < 0 || a->steps < 0 || a->dim < 0 || a->reserved != 0) return MORPH_EINVAL;
  if (a->states < 1 || a->states > MORPH_SSM_MAX_STATES) return MORPH_ERANGE;
  if (!known_dtype(dtype)) return MORPH_EDTYPE;
  if (a->batch > 0 && a->dim > 0 && (!a->A || (a->steps > 0 && (!a->x || !a->dt || !a->B || !a->C)))) return MORPH_EINVAL;
  const int64_t most = MORPH_SSM_MAX_STEP;
  if (a->batch > INT32_MAX || a->steps > INT32_MAX - kT * kW || a->dim > most) return MORPH_ERANGE;
  for (int64_t step : {a->x_step, a->dt_step, a->z ? a->z_step : 0, a->B_step, a->C_step})
    if (step < 0 || step > most) return MORPH_ERANGE;
  const int64_t all = INT64_MAX >> 12;
  if (a->batch > 0 && a->dim > 0 && (a->dim > all / a->batch || a->steps > all / a->batch / a->dim)) return MORPH_ERANGE;
  return MORPH_OK;
}

Scan scan_of(const morph_ssm* a, const Plan& plan, int bytes) {
  auto view = [&](const void* p, int64_t batch, int64_t step) {
    return View{static_cast<const char*>(p), batch * bytes, (int32_t)(step * bytes)};
  };
  Scan s{};
  s.x = view(a->x, a->x_batch, a->x_step), s.dt = view(a->dt, a->dt_batch, a->dt_step);
  s.B = view(a->B, a->B_batch, a->B_step), s.C = view(a->C, a->C_batch, a->C_step);
  if (a->z) s.z = view(a->z, a->z_batch, a->z_step);
  s.A = a->A, s.skip = a->skip, s.dt_bias = a->dt_bias;
  s.batch = (int32_t)a->batch, s.steps = (int32_t)a->steps, s.dim = (int32_t)a->dim, s.states = a->states;
  s.tiles = (int32_t)plan.tiles, s.groups = (int32_t)plan.groups, s.segments = (int32_t)plan.segments;
  s.per = (int32_t)plan.per;
  return s;
}

// What enters each segment, into ends [segments][batch][dim][states].
template <typename T, int L, bool kBack, bool kGated>
int join_segments(const Scan& a, const float* first, float* ends, float* sums, hipStream_t s) {
  if (a.segments < 2) return MORPH_OK;
  const int64_t blocks = (int64_t)a.groups * a.batch * (a.segments - 1);
  auto find = [&](auto waves) {
    constexpr int kWaves = decltype(waves)::value;
    hipLaunchKernelGGL((ssm_ends_kernel<T, L, kBack, kGated && kBack, kWaves>), dim3((unsigned)blocks), dim3(64 * kWaves), 0, s, a,
                       ends, sums);
  };
  if (a.per >= kManyTiles) find(std::integral_constant<int, 16>{});
  else find(std::integral_constant<int, 4>{});
  const int rc = launch_status();
  if (rc != MORPH_OK || a.segments <= kJoined) return rc;
  hipLaunchKernelGGL(ssm_join_kernel<kBack>, dim3((unsigned)over((int64_t)a.batch * a.dim * a.states, 256)), dim3(256), 0, s, a,
                     first, ends, sums);
  return launch_status();
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" size_t morph_ssm_workspace_bytes(int64_t batch, int64_t steps, int64_t dim, int states, int backward) {
  if (batch < 1 || steps < 0 || dim < 1 || states < 1 || states > MORPH_SSM_MAX_STATES) return 0;
  return Plan(batch, steps, dim, states).bytes(backward != 0);
}

extern "C" int morph_ssm_forward(const morph_ssm* a, int dtype, void* y, float* last, float* kept, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (const int rc = check(a, dtype)) return rc;
  if (a->batch == 0 || a->dim == 0) return MORPH_OK;
  if ((a->steps > 0 && !y) || !last) return MORPH_EINVAL;
  const Plan plan(a->batch, a->steps, a->dim, a->states);
  if (a->steps != 1 && plan.bytes(false) > 0 && (!workspace || workspace_bytes < plan.bytes(false))) return MORPH_EWORKSPACE;
  if (!launchable(plan.groups * plan.segments * a->batch, 64 * kW) ||
      !launchable(over(a->batch * a->dim * a->states, 256), 256))
    return MORPH_ERANGE;
  hipStream_t s = as_stream(stream);
  return by_form(dtype, a->states, a->z != nullptr, [&](auto t, auto lanes, auto gated) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    constexpr bool kGated = decltype(gated)::value;
    const Scan scan = scan_of(a, plan, Fmt<T>::bytes);
    if (a->steps == 1) {
      const int64_t groups = over(a->dim, 256 / L), blocks = groups * over(a->batch, kSequences);
      hipLaunchKernelGGL((ssm_one_kernel<T, L>), dim3((unsigned)blocks), dim3(256), 0, s, scan, (int)groups, a->first,
                         static_cast<char*>(y), last, kept);
      return launch_status();
    }
    float* ends = static_cast<float*>(workspace);
    if (const int rc = join_segments<T, L, false, kGated>(scan, a->first, ends, ends + plan.states, s)) return rc;
    hipLaunchKernelGGL((ssm_kernel<T, L, kGated>), dim3((unsigned)(plan.groups * plan.segments * a->batch)), dim3(64 * kW), 0,
                       s, scan, a->first, ends, ends + plan.states, static_cast<char*>(y), last, kept);
    return launch_status();
  });
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
  if (dy_step < 0 || dy_step > MORPH_SSM_MAX_STEP) return MORPH_ERANGE;
  const Plan plan(a->batch, a->steps, a->dim, a->states);
  const size_t need = a->batch > 0 ? plan.bytes(true) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return MORPH_EWORKSPACE;
  const int64_t rows = a->batch * a->steps, sums = over(rows * 8 * lanes_of(a->states), 256);
  const int64_t ends = over(a->dim * a->states, 256);
  if (!launchable(sums, 256) || !launchable(sums + ends, 256) || !launchable(over(a->batch * a->dim * a->states, 256), 256) ||
      !launchable(plan.groups * plan.segments * a->batch, 64 * kW))
    return MORPH_ERANGE;
  SsmParts parts;
  parts.bc = static_cast<float*>(workspace);
  parts.A = parts.bc + plan.bc;
  parts.skip = parts.A + plan.states;
  parts.dt_bias = parts.skip + plan.channels;
  parts.late = parts.dt_bias + plan.channels;
  parts.sums = parts.late + plan.states;
  hipStream_t s = as_stream(stream);
  const int rc = by_form(dtype, a->states, a->z != nullptr, [&](auto t, auto lanes, auto gated) {
    using T = decltype(t);
    constexpr int L = decltype(lanes)::value;
    constexpr bool kGated = decltype(gated)::value;
    if (a->batch == 0) return (int)MORPH_OK;
    Scan scan = scan_of(a, plan, Fmt<T>::bytes);
    scan.dy = View{static_cast<const char*>(dy), dy_batch * Fmt<T>::bytes, (int32_t)(dy_step * Fmt<T>::bytes)};
    if (const int status = join_segments<T, L, true, kGated>(scan, dlast, parts.late, parts.sums, s)) return status;
    hipLaunchKernelGGL((ssm_back_kernel<T, L, kGated>), dim3((unsigned)(plan.blocks * plan.segments * a->batch)),
                       dim3(64 * kW), 0, s, scan, (int)plan.blocks, kept, dlast, *g, parts);
    return launch_status();
  });
  if (rc != MORPH_OK) return rc;
  const int wide = 4 * lanes_of(a->states);
  auto sum = [&](auto t) {
    hipLaunchKernelGGL(ssm_sum_kernel<decltype(t)>, dim3((unsigned)(sums + ends)), dim3(256), 0, s, parts, plan.blocks, rows,
                       wide, plan.segments * a->batch, a->dim, a->states, (int)sums, *g);
    return launch_status();
  };
  return dtype == MORPH_DTYPE_F32 ? sum(F32{}) : dtype == MORPH_DTYPE_F16 ? sum(F16{}) : sum(BF16{});
}
