// Gated linear recurrence (morph_layers.h) and its backward pass: s_t = a_t s_(t-1) + (1 - a_t) v_t
// along the steps of [batch, steps, dim], every channel on its own.
//
// The recurrence of a stretch of steps is s -> A s + S with A the product of its gates and S
// its result from a zero state, and two stretches compose: (A2, S2) after (A1, S1) is
// (A2 A1, A2 S1 + S2).  So a workgroup takes a tile of steps and 128 channels, a lane two
// channels, a wave 16 (backward: 8) consecutive steps, all loaded at once; each wave finds its (A, S) in
// registers, the waves' are joined through LDS, and the second pass over the registers starts from
// the true state.  Every tensor is read and written once.  HBM bounds it: 65536 steps of 3072 channels in
// BF16 with z take 287 us forward (1.61 GB and 13 MB of states, 5.7 TB/s) and 540 us backward (2.82 GB, 5.3 TB/s).
// Steps that fit one wave have a tile of one: 64 sequences of 2 to 16 steps of 3072 channels take
// 7.2 to 8.5 us instead of 13.6 with the seven idle waves.
//
// Tiles of one channel group follow each other in time through memory, with the same sums
// whatever their timing: kRun tiles make a run, kRuns runs a stretch.  A tile publishes its (A, S)
// before it waits for anything, the last tile of a run the run's (A, S) as soon as the run's tiles
// have theirs, the last of a stretch the state behind it.  What enters a tile is the state that its
// stretch begins with, through the (A, S) of the runs and then of the tiles before it, in order.
// (Taking whichever is there, a state or an (A, S), would round differently from call to call.)  So
// only the stretches wait for each other, 0.7 us each time.  Where there are many channel groups a
// stretch is a single run (kManyGroups).
// A published word is 64 bits and tells by itself whether it is there, so no ordering between
// words is needed.  Tiles are taken by ticket, earlier times first: what a tile waits for is always
// running or done, so every wait ends (kSpins bounds it all the same).
//
// The forward applies every step's (A, S) from the tile's beginning to the state that enters
// the tile, so the state behind a tile's last step is, bit for bit, the one that the next tile of
// its run begins with; where all gates are 1 the state stays as it is, however long.
//
// The backward runs the tiles from the last to the first: r_t = w_t + a_(t+1) r_(t+1) is the same
// recurrence in reversed time with the same A, and the states come again from the one that
// the forward kept for each tile, in the same pass.
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

// A step or none: a lane per channel, no workspace and no wait.  64 sequences of 3072 channels in BF16
// with z take 3.0 us, 6.2 us with the call; two steps of them in a tile's one wave take 7.2 us.
template <typename T>
__global__ __launch_bounds__(64) void scan_one_kernel(morph_scan a, void* __restrict__ y, float* __restrict__ last,
                                                      float* __restrict__ states) {
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y, at = b * a.dim + c;
  if (c >= a.dim) return;
  float s = a.s0 ? a.s0[at] : 0.0f;
  if (a.steps) {
    if (states) states[at] = s;
    const Sigmoid g = sigmoid(load1<T>(a.f, b * a.f_batch + c));
    s = __fmaf_rn(g.a, s, g.b * load1<T>(a.v, b * a.v_batch + c));
    float out = s;
    if (a.z) {
      const float z = load1<T>(a.z, b * a.z_batch + c);
      out = s * (z * sigmoid(z).a);
    }
    store1<T>(y, at, out);
  }
  if (last) last[at] = s;
}

template <typename T>
__global__ __launch_bounds__(64) void scan_one_back_kernel(morph_scan a, const float* __restrict__ states,
                                                           const void* __restrict__ dy, int64_t dy_batch,
                                                           const float* __restrict__ dlast, void* __restrict__ df,
                                                           void* __restrict__ dv, void* __restrict__ dz,
                                                           float* __restrict__ ds0) {
  const int64_t c = (int64_t)blockIdx.x * 64 + threadIdx.x, b = blockIdx.y, at = b * a.dim + c;
  if (c >= a.dim) return;
  float r = dlast ? dlast[at] : 0.0f;
  if (a.steps) {
    const float s = states[at], v = load1<T>(a.v, b * a.v_batch + c);
    const Sigmoid g = sigmoid(load1<T>(a.f, b * a.f_batch + c));
    float w = load1<T>(dy, b * dy_batch + c);
    if (a.z) {
      const float z = load1<T>(a.z, b * a.z_batch + c);
      const Sigmoid q = sigmoid(z);
      store1<T>(dz, at, w * __fmaf_rn(g.a, s, g.b * v) * (q.a * __fmaf_rn(z, q.b, 1.0f)));
      w *= z * q.a;
    }
    r += w;
    store1<T>(dv, at, g.b * r);
    store1<T>(df, at, r * (s - v) * (g.a * g.b));
    r *= g.a;
  }
  if (ds0) ds0[at] = r;
}

// ---- tiles ----------------------------------------------------------------------

constexpr int kWaves = 8;  // of a tile; 1 where one wave has all steps
constexpr int kForwardSteps = 16;  // of a wave: 128 steps a tile
constexpr int kBackwardSteps = 8;  // 64: the backward holds four values per step and channel
constexpr int kSpins = 1 << 20;
constexpr int kTicketBytes = 256;
static_assert(kWaves * kBackwardSteps == kSpan, "a backward tile begins with a kept state");
static_assert(kSpan % kForwardSteps == 0, "states are kept at a wave's first step");

// kVec consecutive channels of one step as loaded: 16-bit pairs or singles, floats.
template <typename T, int kVec>
struct Raw {
  typedef std::conditional_t<kVec == 2, uint32_t, uint16_t> type;
};
template <int kVec>
struct Raw<F32, kVec> {
  typedef float type __attribute__((ext_vector_type(kVec)));
};
template <typename T, int kVec>
__device__ __forceinline__ float value(const typename Raw<T, kVec>::type& r, int k) {
  if constexpr (std::is_same_v<T, F32>) return r[k];
  else return to_float<T>(k ? (uint32_t)r >> 16 : r & 0xFFFFu);
}

// The tile's rows of one tensor: a wave-uniform address that advances by the step, and the
// lane's offset in it.  kStream: past the caches (streams() on the host).
template <typename T, int kVec, bool kStream>
struct Rows {
  typedef typename Raw<T, kVec>::type raw;
  const char* at;
  int64_t step;  // bytes
  __device__ __forceinline__ Rows(const void* p, int64_t first, int64_t stride)
      : at(static_cast<const char*>(p) + first * Fmt<T>::bytes), step(stride * Fmt<T>::bytes) {}
  __device__ __forceinline__ raw load(int i, uint32_t lane) const {
    return load_stream<kStream>(reinterpret_cast<const raw*>(at + i * step + lane));
  }
  __device__ __forceinline__ void store(int i, uint32_t lane, const float (&x)[kVec]) const {
    raw v;
    if constexpr (std::is_same_v<T, F32>) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) v[k] = x[k];
    } else if constexpr (kVec == 2) {
      v = pack2<T>(x[0], x[1]);
    } else {
      v = (uint16_t)from_float<T>(x[0]);
    }
    store_stream<kStream>(reinterpret_cast<raw*>(const_cast<char*>(at) + i * step + lane), v);
  }
};

// A launch's tiles: `groups` = batch x channel groups, `tiles` steps' tiles of each.
struct ScanGrid {
  uint32_t* ticket;  // the workspace: tickets given out, then
  uint64_t* parts;   // [tiles][groups][64 lanes][kVec]: A, S
  uint64_t* runs;    // [runs][groups][64 lanes][kVec]: A, S
  uint64_t* states;  // [stretches][groups][64 lanes][kVec]: what stretch 1, 2, ... begins with, twice
  int32_t tiles, groups, channel_groups;
  int32_t in_stretch;  // runs of a stretch: kRuns or 1
};
constexpr int kRun = 8;   // tiles of a run: a word of one for each wave to fetch
constexpr int kRuns = 8;  // runs of a stretch, likewise
static_assert(kRun <= kWaves && kRuns <= kWaves,
              "the last wave, which fetches the stretch's first state, has no tile's or run's words to fetch");
constexpr uint64_t kNothing = ~uint64_t(0);  // a word that is not published yet

// Two floats as one word.  A pair of NaN that reads as kNothing loses a bit of its payload, so that it
// is not waited for.
__device__ __forceinline__ void publish(uint64_t* at, float x, float y) {
  const uint64_t w = ((uint64_t)__builtin_bit_cast(uint32_t, y) << 32) | __builtin_bit_cast(uint32_t, x);
  __hip_atomic_store(at, w == kNothing ? w ^ 1 : w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// kCount words of this lane, once all of the wave's are published (NaN should that never be).
template <int kCount>
__device__ __forceinline__ void fetch(const uint64_t* at, float (&x)[kCount], float (&y)[kCount]) {
  uint64_t w[kCount];
  bool all = false;
  for (int spin = 0; spin < kSpins && !all; ++spin) {
    bool mine = true;
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      w[i] = __hip_atomic_load(at + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      mine = mine && w[i] != kNothing;
    }
    all = __all(mine);
  }
#pragma unroll
  for (int i = 0; i < kCount; ++i) {
    x[i] = all ? __builtin_bit_cast(float, (uint32_t)w[i]) : __builtin_nanf("");
    y[i] = all ? __builtin_bit_cast(float, (uint32_t)(w[i] >> 32)) : __builtin_nanf("");
  }
}

// This workgroup's tile, in the order of the tickets, and its group.
__device__ __forceinline__ int take_tile(const ScanGrid& g, int& group) {
  int id = (int)blockIdx.x;
  if (g.tiles > 1) {
    __shared__ int mine;
    if (threadIdx.x == 0)
      mine = (int)__hip_atomic_fetch_add(g.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    id = mine;
  }
  id = __builtin_amdgcn_readfirstlane(id);
  group = id % g.groups;
  return id / g.groups;
}

// The way of a tile's state through its waves and to the next tile, in two steps with room for
// work between them: start() publishes the tile's (A, S) as soon as its waves have met, and by
// finish() the (A, S) of the tiles before have mostly arrived.  `order`: the wave's place in the
// direction of the walk.
template <int kW, int kVec>
struct Entering {
  float wa[kVec], ws[kVec];  // (A, S) of the tile's steps before this wave
  float la[kVec], ls[kVec];  // with this wave's: of the whole tile in the last one
  float carry[kVec];         // what enters the tile

  // Adds a wave's (A, S), and with kBack the backward's states' sums T over the same gates, whose
  // walk is the other way: `state` goes from what enters the tile to what enters the wave.
  template <bool kBack>
  __device__ __forceinline__ void start(const ScanGrid& g, int tile, int group, int order, int lane,
                                        const float (&A)[kVec], const float (&S)[kVec], const float (&T)[kVec],
                                        float (&state)[kVec]) {
    __shared__ float sa[kW][kVec][64], ss[kW][kVec][64], st[kBack ? kW : 1][kVec][64];
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      sa[order][k][lane] = A[k], ss[order][k][lane] = S[k];
      if constexpr (kBack) st[order][k][lane] = T[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      wa[k] = 1.0f, ws[k] = 0.0f;
      for (int w = 0; w < order; ++w) {
        ws[k] = __fmaf_rn(sa[w][k][lane], ws[k], ss[w][k][lane]);
        wa[k] *= sa[w][k][lane];
      }
      ls[k] = __fmaf_rn(A[k], ws[k], S[k]), la[k] = wa[k] * A[k];
    }
    const int before = tile % kRun;
    if (g.tiles > 1 && order == kW - 1 && before < kRun - 1 && tile + 1 < g.tiles) {
      const int64_t mine = ((int64_t)group * 64 + lane) * kVec, stride = (int64_t)g.groups * 64 * kVec;
#pragma unroll
      for (int k = 0; k < kVec; ++k) publish(g.parts + tile * stride + mine + k, la[k], ls[k]);
    }
    if constexpr (kBack) {
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        for (int w = kW - 1; w > order; --w) state[k] = __fmaf_rn(sa[w][k][lane], state[k], st[w][k][lane]);
    }
  }

  // first: this lane's share of what enters the first tile, read in the first stretch; null: zero.
  __device__ __forceinline__ void finish(const ScanGrid& g, int tile, int group, int order, int lane,
                                         const float* first) {
    __shared__ float pa[kRun][kVec][64], ps[kRun][kVec][64];    // the run's tiles
    __shared__ float qa[kRuns][kVec][64], qs[kRuns][kVec][64];  // the stretch's runs
    __shared__ float begin[kVec][64];
    if (kW < kWaves || g.tiles == 1) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) carry[k] = first ? first[k] : 0.0f;
      return;
    }
    const int run = tile / kRun, before = tile % kRun;
    const int stretch = g.in_stretch > 1 ? run / kRuns : run, earlier = g.in_stretch > 1 ? run % kRuns : 0;
    const int64_t mine = ((int64_t)group * 64 + lane) * kVec, stride = (int64_t)g.groups * 64 * kVec;
    float x[kVec], y[kVec];
    if (order < before) {
      fetch<kVec>(g.parts + ((int64_t)run * kRun + order) * stride + mine, x, y);
#pragma unroll
      for (int k = 0; k < kVec; ++k) pa[order][k][lane] = x[k], ps[order][k][lane] = y[k];
    }
    if (before == kRun - 1 && earlier < g.in_stretch - 1 && tile + 1 < g.tiles) {
      __syncthreads();
      if (order == kW - 1) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          float A = 1.0f, S = 0.0f;
          for (int i = 0; i < before; ++i) S = __fmaf_rn(pa[i][k][lane], S, ps[i][k][lane]), A *= pa[i][k][lane];
          publish(g.runs + run * stride + mine + k, A * la[k], __fmaf_rn(la[k], S, ls[k]));
        }
      }
    }
    if (order < earlier) {
      fetch<kVec>(g.runs + ((int64_t)stretch * kRuns + order) * stride + mine, x, y);
#pragma unroll
      for (int k = 0; k < kVec; ++k) qa[order][k][lane] = x[k], qs[order][k][lane] = y[k];
    }
    if (order == kW - 1) {
      if (stretch > 0) {
        fetch<kVec>(g.states + stretch * stride + mine, x, y);
      } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k) x[k] = first ? first[k] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kVec; ++k) begin[k][lane] = x[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      carry[k] = begin[k][lane];
      for (int i = 0; i < earlier; ++i) carry[k] = __fmaf_rn(qa[i][k][lane], carry[k], qs[i][k][lane]);
      for (int i = 0; i < before; ++i) carry[k] = __fmaf_rn(pa[i][k][lane], carry[k], ps[i][k][lane]);
    }
    if (order == kW - 1 && before == kRun - 1 && earlier == g.in_stretch - 1 && tile + 1 < g.tiles) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        const float next = __fmaf_rn(la[k], carry[k], ls[k]);
        publish(g.states + (stretch + 1) * stride + mine + k, next, next);
      }
    }
  }
};

// A wave's place: its tile's group, channels and steps.
template <typename T, int kW, int kVec>
struct Place {
  int64_t b, channel, c, t0;  // channel: the group's first; c: the lane's first
  int n;                      // steps, <= 0: none
  uint32_t lane;              // bytes
  bool active;
  __device__ __forceinline__ Place(const morph_scan& a, const ScanGrid& g, int tile, int group, int wave, int L) {
    b = group / g.channel_groups;
    channel = (int64_t)(group % g.channel_groups) * 64 * kVec;
    const int l = threadIdx.x & 63;
    active = channel + l * kVec < a.dim;
    const int own = active ? l * kVec : 0;  // lanes past the end repeat the first and store nothing
    c = channel + own;
    lane = (uint32_t)own * Fmt<T>::bytes;
    t0 = ((int64_t)tile * kW + wave) * L;
    n = (int)(a.steps - t0 < L ? a.steps - t0 : L);
  }
};

// Runs body(std::true_type) where the wave has all its steps, else body(std::false_type): the
// tests for the sequence's end are in the second form only.
template <typename F>
__device__ __forceinline__ void whole_or_part(bool whole, F&& body) {
  if (whole) body(std::true_type{});
  else body(std::false_type{});
}

template <typename T, int kW, int kVec, bool kGated, bool kStream>
__global__ __launch_bounds__(64 * kW, 4) void scan_tile_kernel(const morph_scan a, const ScanGrid g,
                                                             void* __restrict__ y, float* __restrict__ last,
                                                             float* __restrict__ states) {
  static_assert(kVec == 2 || !kStream, "what by_form asks for");
  constexpr int L = kForwardSteps;
  typedef typename Raw<T, kVec>::type raw;
  int group;
  const int tile = take_tile(g, group);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place<T, kW, kVec> p(a, g, tile, group, wave, L);

  float A[kVec], S[kVec], pa[L][kVec], ps[L][kVec];  // (A, S) from the wave's first step on
  raw z[kGated ? L : 1];
#pragma unroll
  for (int k = 0; k < kVec; ++k) A[k] = 1.0f, S[k] = 0.0f;
  const Rows<T, kVec, kStream> rf(a.f, p.b * a.f_batch + p.t0 * a.f_step + p.channel, a.f_step);
  const Rows<T, kVec, kStream> rv(a.v, p.b * a.v_batch + p.t0 * a.v_step + p.channel, a.v_step);
  const Rows<T, kVec, kStream> rz(a.z, p.b * a.z_batch + p.t0 * a.z_step + p.channel, a.z_step);
  if (p.n > 0) {
    whole_or_part(p.n == L, [&](auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      raw f[L], v[L];
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int j = kWhole || i < p.n ? i : p.n - 1;
        f[i] = rf.load(j, p.lane);
        v[i] = rv.load(j, p.lane);
      }
      if constexpr (kGated) {
#pragma unroll
        for (int i = 0; i < L; ++i) z[i] = rz.load(kWhole || i < p.n ? i : p.n - 1, p.lane);
      }
#pragma unroll
      for (int i = 0; i < L; ++i) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          const Sigmoid s = sigmoid(value<T, kVec>(f[i], k));
          float gate = s.a, in = s.b * value<T, kVec>(v[i], k);
          if (!kWhole && i >= p.n) gate = 1.0f, in = 0.0f;  // steps past the end pass the state on
          ps[i][k] = S[k] = __fmaf_rn(gate, S[k], in);
          pa[i][k] = A[k] *= gate;
        }
      }
    });
  }
  float none[kVec];
  Entering<kW, kVec> e;
  e.template start<false>(g, tile, group, wave, threadIdx.x & 63, A, S, A, none);
  float act[kGated ? L : 1][kVec];  // silu(z), while the tiles before publish
  if constexpr (kGated) {
    if (p.n > 0) {
#pragma unroll
      for (int i = 0; i < L; ++i)
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          const float q = value<T, kVec>(z[i], k);
          act[i][k] = q * gate_sigmoid(q);
        }
    }
  }
  e.finish(g, tile, group, wave, threadIdx.x & 63, a.s0 ? a.s0 + (p.b * a.dim + p.c) : nullptr);
  if (!p.active || p.n <= 0) return;
  if (states && p.t0 % kSpan == 0) {
    const int64_t spans = (a.steps + kSpan - 1) / kSpan;
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      states[(p.b * spans + p.t0 / kSpan) * a.dim + p.c + k] = __fmaf_rn(e.wa[k], e.carry[k], e.ws[k]);
  }
  const Rows<T, kVec, kStream> ry(y, (p.b * a.steps + p.t0) * a.dim + p.channel, a.dim);
  whole_or_part(p.n == L, [&](auto whole) {
    float s[kVec];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      float out[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        s[k] = out[k] = __fmaf_rn(e.wa[k] * pa[i][k], e.carry[k], __fmaf_rn(pa[i][k], e.ws[k], ps[i][k]));
        if constexpr (kGated) out[k] *= act[i][k];
      }
      if (decltype(whole)::value || i < p.n) ry.store(i, p.lane, out);
    }
    if (last && p.t0 + p.n == a.steps) {
#pragma unroll
      for (int k = 0; k < kVec; ++k) last[p.b * a.dim + p.c + k] = s[k];
    }
  });
}

template <typename T, int kW, int kVec, bool kGated, bool kStream>
__global__ __launch_bounds__(64 * kW, 4) void scan_tile_back_kernel(const morph_scan a, const ScanGrid g,
                                                                  const float* __restrict__ states,
                                                                  const void* __restrict__ dy, int64_t dy_batch,
                                                                  int64_t dy_step, const float* __restrict__ dlast,
                                                                  void* __restrict__ df, void* __restrict__ dv,
                                                                  void* __restrict__ dz, float* __restrict__ ds0) {
  static_assert(kVec == 2 || !kStream, "what by_form asks for");
  constexpr int L = kBackwardSteps;
  typedef typename Raw<T, kVec>::type raw;
  int group;
  const int walked = take_tile(g, group);
  const int tile = g.tiles - 1 - walked;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place<T, kW, kVec> p(a, g, tile, group, wave, L);

  // gate: a; pass: 1 - a; w: dy silu(z); x: v, then what r is multiplied by for df
  float gate[L][kVec], pass[L][kVec], w[L][kVec], x[L][kVec], slope[kGated ? L : 1][kVec];
  float A[kVec], S[kVec], R[kVec], s[kVec], r[kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k) A[k] = 1.0f, S[k] = 0.0f, R[k] = 0.0f;
  const Rows<T, kVec, kStream> rf(a.f, p.b * a.f_batch + p.t0 * a.f_step + p.channel, a.f_step);
  const Rows<T, kVec, kStream> rv(a.v, p.b * a.v_batch + p.t0 * a.v_step + p.channel, a.v_step);
  const Rows<T, kVec, kStream> rz(a.z, p.b * a.z_batch + p.t0 * a.z_step + p.channel, a.z_step);
  {
    const int64_t spans = (a.steps + kSpan - 1) / kSpan;
#pragma unroll
    for (int k = 0; k < kVec; ++k) s[k] = states[(p.b * spans + tile) * a.dim + p.c + k];
  }
  const Rows<T, kVec, kStream> rd(dy, p.b * dy_batch + p.t0 * dy_step + p.channel, dy_step);
  if (p.n > 0) {
    whole_or_part(p.n == L, [&](auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      raw f[L], v[L], z[kGated ? L : 1], d[L];
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const int j = kWhole || i < p.n ? i : p.n - 1;
        f[i] = rf.load(j, p.lane);
        v[i] = rv.load(j, p.lane);
        if constexpr (kGated) z[i] = rz.load(j, p.lane);
        d[i] = rd.load(j, p.lane);
      }
#pragma unroll
      for (int i = 0; i < L; ++i) {
        const bool inside = kWhole || i < p.n;
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          const Sigmoid q = sigmoid(value<T, kVec>(f[i], k));
          gate[i][k] = inside ? q.a : 1.0f;
          pass[i][k] = inside ? q.b : 0.0f;
          x[i][k] = inside ? value<T, kVec>(v[i], k) : 0.0f;
          w[i][k] = inside ? value<T, kVec>(d[i], k) : 0.0f;
          if constexpr (kGated) {
            const Silu h = silu(inside ? value<T, kVec>(z[i], k) : 0.0f);
            slope[i][k] = w[i][k] * h.slope;
            w[i][k] *= h.y;
          }
          S[k] = __fmaf_rn(gate[i][k], S[k], pass[i][k] * x[i][k]);
          A[k] *= gate[i][k];
        }
      }
    });
#pragma unroll
    for (int i = L - 1; i >= 0; --i)
#pragma unroll
      for (int k = 0; k < kVec; ++k) R[k] = gate[i][k] * (w[i][k] + R[k]);
  }
  const int order = kW - 1 - wave;
  Entering<kW, kVec> e;
  e.template start<true>(g, walked, group, order, lane, A, R, S, s);
  const int64_t at = (p.b * a.steps + p.t0) * a.dim + p.channel;
  if (p.n > 0) {
    const Rows<T, kVec, kStream> oz(dz, at, a.dim);
    whole_or_part(p.n == L, [&](auto whole) {
#pragma unroll
      for (int i = 0; i < L; ++i) {
        float out[kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          const float prev = s[k], v = x[i][k];
          s[k] = __fmaf_rn(gate[i][k], prev, pass[i][k] * v);
          x[i][k] = (prev - v) * (gate[i][k] * pass[i][k]);
          if constexpr (kGated) out[k] = slope[i][k] * s[k];
        }
        if constexpr (kGated)
          if ((decltype(whole)::value || i < p.n) && p.active) oz.store(i, p.lane, out);
      }
    });
  }
  e.finish(g, walked, group, order, lane, dlast ? dlast + (p.b * a.dim + p.c) : nullptr);
  if (!p.active || p.n <= 0) return;
#pragma unroll
  for (int k = 0; k < kVec; ++k) r[k] = __fmaf_rn(e.wa[k], e.carry[k], e.ws[k]);
  const Rows<T, kVec, kStream> of(df, at, a.dim), ov(dv, at, a.dim);
  whole_or_part(p.n == L, [&](auto whole) {
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
      float gf[kVec], gv[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        r[k] += w[i][k];
        gv[k] = r[k] * pass[i][k];
        gf[k] = r[k] * x[i][k];
        r[k] *= gate[i][k];
      }
      if (decltype(whole)::value || i < p.n) {
        ov.store(i, p.lane, gv);
        of.store(i, p.lane, gf);
      }
    }
  });
  if (ds0 && p.t0 == 0) {
#pragma unroll
    for (int k = 0; k < kVec; ++k) ds0[p.b * a.dim + p.c + k] = r[k];
  }
}

// The tickets (zero) and words (kNothing) of a launch.  (A kernel, not a memset: a captured memset node is
// not replayed reliably.)
__global__ __launch_bounds__(256) void scan_clear_kernel(u32x4* p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t x = i < kTicketBytes / 16 ? 0u : 0xFFFFFFFFu;
  if (i < n) p[i] = u32x4{x, x, x, x};
}

bool float_type(int dtype) {
  return dtype == MORPH_DTYPE_F32 || dtype == MORPH_DTYPE_F16 || dtype == MORPH_DTYPE_BF16;
}

int scan_check(const morph_scan* a, int dtype) {
  if (a == nullptr || a->batch < 0 || a->steps < 0 || a->dim < 0) return MORPH_EINVAL;
  if (!float_type(dtype)) return MORPH_EDTYPE;
  if (a->batch > 65535 || a->dim > (int64_t(1) << 30) || a->steps > (int64_t(1) << 40))
    return MORPH_ERANGE;
  // every offset, byte count and tile count below fits 64 bits
  int64_t rows;
  if (__builtin_mul_overflow(a->batch, a->steps, &rows) || (a->dim > 0 && rows > (int64_t(1) << 46) / a->dim))
    return MORPH_ERANGE;
  if (a->batch && a->steps && a->dim && (a->f == nullptr || a->v == nullptr)) return MORPH_EINVAL;
  return MORPH_OK;
}

// ---- host -------------------------------------------------------------------------

int64_t tiles_of(int64_t steps, bool backward) {
  const int64_t span = kWaves * (backward ? kBackwardSteps : kForwardSteps);
  return (steps + span - 1) / span;
}
// Words for either channel count per lane, channels rounded up to 128: one a tile, a run and a stretch.
int64_t runs_of(int64_t tiles) { return (tiles + kRun - 1) / kRun; }
size_t scan_words(int64_t channels, int64_t tiles) {
  return (size_t)channels * (size_t)(tiles + 2 * runs_of(tiles));
}
size_t scan_workspace(int64_t batch, int64_t steps, int64_t dim, bool backward) {
  const int64_t tiles = tiles_of(steps, backward);
  if (batch <= 0 || dim <= 0 || tiles <= 1) return 0;
  return kTicketBytes + 8 * scan_words(batch * ((dim + 127) / 128 * 128), tiles);
}

// Whether all of a tensor's rows begin at multiples of `bytes`.
bool starts(const void* p, int64_t batch, int64_t step, int64_t size, int64_t bytes) {
  return p == nullptr ||
         (batch * size % bytes == 0 && step * size % bytes == 0 && reinterpret_cast<uintptr_t>(p) % bytes == 0);
}
constexpr int64_t kLine = 128;

// From so many channel groups on a stretch is one run: few of the resident workgroups then belong to one
// group and wait for each other, and the runs' words cost more than the waits.  Measured, us, stretches of 1 / 8 runs,
// forward and backward of 65536 steps in BF16 with z: 24 groups 820 / 837, 16 566 / 577, 12 455 / 446,
// 8 358 / 317; forward of 2 x 30574 x 238 (4 groups) 64 / 43.
constexpr int64_t kManyGroups = 16;

int scan_grid(const morph_scan* a, int waves, int kvec, bool backward, void* workspace, hipStream_t s, ScanGrid& g,
              unsigned& grid) {
  const int64_t groups_c = (a->dim + 64 * kvec - 1) / (64 * kvec), groups = groups_c * a->batch;
  const int64_t tiles = tiles_of(a->steps, backward), total = tiles * groups;
  if (!launchable(total, 64 * waves)) return MORPH_ERANGE;
  g.ticket = static_cast<uint32_t*>(workspace);
  g.parts = reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + kTicketBytes);
  g.runs = g.parts + total * 64 * kvec;
  g.states = g.runs + runs_of(tiles) * groups * 64 * kvec;
  g.in_stretch = groups < kManyGroups ? kRuns : 1;
  g.tiles = (int32_t)tiles, g.groups = (int32_t)groups, g.channel_groups = (int32_t)groups_c;
  grid = (unsigned)total;
  if (tiles > 1) {
    const int64_t n = (int64_t)(kTicketBytes + 8 * scan_words(groups * 64 * kvec, tiles)) / 16;
    hipLaunchKernelGGL(scan_clear_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s,
                       static_cast<u32x4*>(workspace), n);
  }
  return MORPH_OK;
}

// Whether a call's tensors are more than the Infinity Cache holds (256 MB), so that what is read and
// written past the caches loses nothing to whoever comes next.  Measured, us, ordinary / past
// the caches, BF16 with z: forward and backward of 65536 x 3072 341 / 293 and 632 / 545, of
// 8 x 4096 x 3072 156 / 150 and 297 / 268; of 4 x 1024 x 3072 (100 and 176 MB, partly in the
// cache from the kernel before) 31.0 / 31.4 and 45 / 48.  Not where a channel group's rows end within a cache
// line, which two groups then share: forward and backward of 20 x 2694 steps, FP16 with z, 2048 channels
// 528 / 484, 2040 635 / 769, 2032 615 / 648; 7 x 6200 x 2200 in FP32 936 / 1015.
bool streams(const morph_scan* a, int dtype, bool backward, bool lines) {
  const int64_t tensors = (a->z != nullptr ? 3 : 2) * (backward ? 2 : 1) + 1;
  return lines && a->batch * a->steps * a->dim * tensors * (dtype == MORPH_DTYPE_F32 ? 4 : 2) > (int64_t(256) << 20);
}

// A call's kernel by its types: F(T, waves a tile, channels a lane, output gate, streams).  What streams has two
// channels a lane: its rows are whole cache lines.
template <typename F>
void by_form(int dtype, bool one_wave, bool two, bool gated, bool stream, F&& f) {
  auto with = [&](auto type, auto waves, auto past) {
    auto lanes = [&](auto channels) {
      if (gated) f(type, waves, channels, std::true_type{}, past);
      else f(type, waves, channels, std::false_type{}, past);
    };
    if constexpr (decltype(past)::value) lanes(std::integral_constant<int, 2>{});
    else if (two) lanes(std::integral_constant<int, 2>{});
    else lanes(std::integral_constant<int, 1>{});
  };
  auto typed = [&](auto waves, auto past) {
    if (dtype == MORPH_DTYPE_F32) with(F32{}, waves, past);
    else if (dtype == MORPH_DTYPE_F16) with(F16{}, waves, past);
    else with(BF16{}, waves, past);
  };
  if (one_wave) typed(std::integral_constant<int, 1>{}, std::false_type{});
  else if (stream) typed(std::integral_constant<int, kWaves>{}, std::true_type{});
  else typed(std::integral_constant<int, kWaves>{}, std::false_type{});
}

}  // namespace
}  // namespace morph

using namespace morph;

extern "C" size_t morph_scan_workspace_bytes(int64_t batch, int64_t steps, int64_t dim, int, int backward) {
  return scan_workspace(batch, steps, dim, backward != 0);
}

extern "C" int morph_scan_forward(const morph_scan* scan, int dtype, void* y, float* last, float* states,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  const int status = scan_check(scan, dtype);
  if (status != MORPH_OK) return status;
  if (scan->batch == 0 || scan->dim == 0) return MORPH_OK;
  if (scan->steps > 0 && y == nullptr) return MORPH_EINVAL;
  const size_t need = scan_workspace(scan->batch, scan->steps, scan->dim, false);
  if (need > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < need))
    return MORPH_EWORKSPACE;
  hipStream_t s = as_stream(stream);
  const morph_scan a = *scan;
  if (a.steps <= 1) {
    const dim3 grid((unsigned)((a.dim + 63) / 64), (unsigned)a.batch);
    by_form(dtype, true, false, false, false, [&](auto type, auto, auto, auto, auto) {
      hipLaunchKernelGGL(scan_one_kernel<decltype(type)>, grid, dim3(64), 0, s, a, y, last, states);
    });
    return launch_status();
  }
  const int64_t size = dtype == MORPH_DTYPE_F32 ? 4 : 2;
  auto all = [&](int64_t bytes) {
    return a.dim * size % bytes == 0 && starts(a.f, a.f_batch, a.f_step, size, bytes) &&
           starts(a.v, a.v_batch, a.v_step, size, bytes) && starts(a.z, a.z_batch, a.z_step, size, bytes) &&
           starts(y, 0, 0, size, bytes);
  };
  const bool two = all(2 * size);  // channels a lane
  const bool one_wave = a.steps <= kForwardSteps;
  ScanGrid g;
  unsigned grid;
  const int shape = scan_grid(scan, one_wave ? 1 : kWaves, two ? 2 : 1, false, workspace, s, g, grid);
  if (shape != MORPH_OK) return shape;
  auto launch = [&](auto type, auto waves, auto vec, auto gated, auto past) {
    hipLaunchKernelGGL((scan_tile_kernel<decltype(type), decltype(waves)::value, decltype(vec)::value,
                                         decltype(gated)::value, decltype(past)::value>),
                       dim3(grid), dim3(64 * decltype(waves)::value), 0, s, a, g, y, last, states);
  };
  by_form(dtype, one_wave, two, a.z != nullptr, streams(scan, dtype, false, all(kLine)), launch);
  return launch_status();
}

extern "C" int morph_scan_backward(const morph_scan* scan, int dtype, const float* states, const void* dy,
                                   int64_t dy_batch, int64_t dy_step, const float* dlast, void* df, void* dv,
                                   void* dz, float* ds0, void* workspace, size_t workspace_bytes, void* stream) {
  const int status = scan_check(scan, dtype);
  if (status != MORPH_OK) return status;
  if (scan->batch == 0 || scan->dim == 0) return MORPH_OK;
  if (scan->steps > 0 && (states == nullptr || dy == nullptr || df == nullptr || dv == nullptr ||
                          (scan->z != nullptr && dz == nullptr)))
    return MORPH_EINVAL;
  const size_t need = scan_workspace(scan->batch, scan->steps, scan->dim, true);
  if (need > 0 && (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < need))
    return MORPH_EWORKSPACE;
  hipStream_t s = as_stream(stream);
  const morph_scan a = *scan;
  if (a.steps <= 1) {
    const dim3 grid((unsigned)((a.dim + 63) / 64), (unsigned)a.batch);
    by_form(dtype, true, false, false, false, [&](auto type, auto, auto, auto, auto) {
      hipLaunchKernelGGL(scan_one_back_kernel<decltype(type)>, grid, dim3(64), 0, s, a, states, dy, dy_batch,
                         dlast, df, dv, dz, ds0);
    });
    return launch_status();
  }
  const int64_t size = dtype == MORPH_DTYPE_F32 ? 4 : 2;
  auto all = [&](int64_t bytes) {
    return a.dim * size % bytes == 0 && starts(a.f, a.f_batch, a.f_step, size, bytes) &&
           starts(a.v, a.v_batch, a.v_step, size, bytes) && starts(a.z, a.z_batch, a.z_step, size, bytes) &&
           starts(dy, dy_batch, dy_step, size, bytes) && starts(df, 0, 0, size, bytes) &&
           starts(dv, 0, 0, size, bytes) && starts(dz, 0, 0, size, bytes);
  };
  const bool two = all(2 * size);  // channels a lane
  const bool one_wave = a.steps <= kBackwardSteps;
  ScanGrid g;
  unsigned grid;
  const int shape = scan_grid(scan, one_wave ? 1 : kWaves, two ? 2 : 1, true, workspace, s, g, grid);
  if (shape != MORPH_OK) return shape;
  auto launch = [&](auto type, auto waves, auto vec, auto gated, auto past) {
    hipLaunchKernelGGL((scan_tile_back_kernel<decltype(type), decltype(waves)::value, decltype(vec)::value,
                                         decltype(gated)::value, decltype(past)::value>),
                       dim3(grid), dim3(64 * decltype(waves)::value), 0, s, a, g, states, dy, dy_batch, dy_step, dlast,
                       df, dv, dz, ds0);
  };
  by_form(dtype, one_wave, two, a.z != nullptr, streams(scan, dtype, true, all(kLine)), launch);
  return launch_status();
}
