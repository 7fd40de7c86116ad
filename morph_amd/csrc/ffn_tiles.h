// The products of the gated feed-forward block on gfx950 MFMA: one workgroup per tile of the
// output, operands through LDS.
//
// Operands.  An operand is stored with K along its rows ("rows": P [M, K], Q [N, K]) or
// across them ("cols": P [K, M], Q [K, N]), so the block's seven products need no transposed
// copy: gate and up and down forward rows . rows, dh and dx rows . cols, the weight
// gradients cols . cols.  Fragments of a "cols" operand come from LDS through gfx950's
// transposing reads.
//
// Tiling and pipeline are the Newton-Schulz products' (gemm.hip, where the constants were
// measured): a tile of 256 x 256 (or 256 x 128, or 128 x 128 with two workgroups per CU, or 64 x 64,
// three with a pipeline of whole stages, where those fill the chip better), four waves with a quarter each
// as 32 x 32 x 16 MFMAs, K in stages of 64, a ring of five LDS slots that hold the P or the Q of one stage, filled by direct loads
// two stages ahead, two register sets of fragments; one barrier per stage.  Every 16-byte
// chunk of an LDS row is stored XOR-swizzled, chosen by which chunk each lane fetches.
//
// Few tiles.  Where an output has fewer tiles than the chip has room for, workgroups of the small shapes take parts
// of K, and their FP32 sums are joined in order by a launch of their own (ffn.hip).
//
// Ragged sizes.  Every load goes through a buffer descriptor that ends with the operand, and
// the hardware gives zeros beyond it: rows past M or N, and for a "cols" operand the rows past K.
// A "rows" operand's chunks past K lie inside the buffer (in the next row), so in the last stage
// of K their offsets are moved out of range by their sign bit.  Both operands are
// therefore zero past K, and what is infinite there meets no zero.  Columns of a "cols"
// operand past M or N hold the next row's values, and reach only outputs that are
// not stored.
//
// Accumulators.  The Q fragment is the MFMA's first operand, so register r of lane (fh, fr) is
// element (row fr, column 8 (r / 4) + 4 fh + r % 4) of a 32 x 32 block: four consecutive columns of
// a row per four registers.  v_permlane32_swap joins them to 16 consecutive columns per lane,
// so 16-bit results leave as 16-byte stores straight from the registers.
#pragma once

#include <algorithm>

#include "ffn.h"

namespace morph {

constexpr int kFfnThreads = 256;

// One output of a launch: C [M, N] (kStore) or the gate's buffers, with its operands.
struct FfnTileProblem {
  const uint16_t* P[2];
  const uint16_t* Q[2];
  uint16_t* C;
  int64_t ldp[2], ldq[2], ldc;
  int32_t M, N;
  int32_t tiles_m, tiles_n;
  int32_t first;   // the launch's first tile of this output
  int32_t vector;  // rows of C allow 16-byte stores
};

constexpr int kFfnProblems = 3;
struct FfnTileArgs {
  FfnTileProblem p[kFfnProblems];
  int32_t count;
  int32_t K;         // of each segment
  int32_t total;     // tiles
  int32_t splits;    // parts of K, of one workgroup each (small tiles of one output; else 1)
  float* parts;      // [splits][M][tiles_n tiles' columns]: their sums, where there are several
  uint16_t *dg, *du;
  void *g, *u;
  uint8_t *g_exponents, *u_exponents;
};

template <int TM, int TN>
struct FfnTile {
  static_assert((TM == 256 || TM == 128 || TM == 64) && (TN == TM || (TM == 256 && TN == 128)), "tile shapes");
  static constexpr int kDepth = 64;                  // K per stage: one 128-byte line per row
  static constexpr int kSlots = TM == 64 ? 6 : 5;    // of the LDS ring; 64: three whole stages
  static constexpr int kSlot = TM * kDepth;          // 16-bit values of a slot: the P or the Q of a stage
  static constexpr int kSmem = kSlots * kSlot;       // 160, 80 or 48 KiB
  static constexpr int kPerCu = TM == 256 ? 1 : TM == 128 ? 2 : 3;  // workgroups per CU
  static constexpr int kBi = TM / 64, kBj = TN / 64;  // 32-wide blocks per wave and dimension
};

typedef __attribute__((address_space(3))) void lds_void;

// ---- epilogues ----------------------------------------------------------------

// a.hi <-> b.lo: the upper 32 lanes of a with the lower 32 of b.
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}

// x: a 32 x 32 block's registers of this lane.  lo and hi: its row's columns 16 fh .. + 7 and
// 16 fh + 8 .. + 15, rounded to T.
template <typename T>
__device__ __forceinline__ void row_words(const float (&x)[16], u32x4& lo, u32x4& hi) {
  uint32_t w[4][2];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    w[q][0] = pack2<T>(x[4 * q], x[4 * q + 1]);
    w[q][1] = pack2<T>(x[4 * q + 2], x[4 * q + 3]);
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    swap_halves(w[0][k], w[2][k]);
    swap_halves(w[1][k], w[3][k]);
  }
  lo = u32x4{w[0][0], w[0][1], w[2][0], w[2][1]};
  hi = u32x4{w[1][0], w[1][1], w[3][0], w[3][1]};
}

template <typename T>
__device__ __forceinline__ void store_row(uint16_t* at, const float (&x)[16]) {
  u32x4 lo, hi;
  row_words<T>(x, lo, hi);
  *reinterpret_cast<u32x4*>(at) = lo;
  *reinterpret_cast<u32x4*>(at + 8) = hi;
}

// Keep a 32 x 32 block of g or u: `at` is the index of its row's first column.
template <int kKeep>
__device__ __forceinline__ void keep_block(const float (&x)[16], void* buffer, uint8_t* exponents,
                                           int64_t at, int fh, bool inside) {
  if constexpr (kKeep == MORPH_FFN_KEEP_FULL) {
    if (!inside) return;
    float* p = static_cast<float*>(buffer) + at + 4 * fh;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(p + 8 * q) = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
  } else if constexpr (kKeep == MORPH_FFN_KEEP_ACT8) {
    uint32_t w[4];
    const int e = act_encode<16>(x, w, [](uint32_t m) {
      uint32_t other = m;  // of the row's other half
      swap_halves(m, other);
      return max(m, other);
    });
    swap_halves(w[0], w[2]);
    swap_halves(w[1], w[3]);
    if (!inside) return;
    *reinterpret_cast<u32x4*>(static_cast<uint8_t*>(buffer) + at + 16 * fh) = u32x4{w[0], w[2], w[1], w[3]};
    if (fh == 0) exponents[at / MORPH_ACT_GROUP] = (uint8_t)e;
  }
}

// A block of g or u as it was kept, loaded ahead of its use.
template <int kKeep>
struct KeptBlock {
  f32x4 v[4];
};
template <>
struct KeptBlock<MORPH_FFN_KEEP_ACT8> {
  u32x4 codes;
  uint32_t exponent;
};
template <int kKeep>
__device__ __forceinline__ void load_kept(KeptBlock<kKeep>& k, const void* buffer, const uint8_t* exponents,
                                          int64_t at, int fh) {
  if constexpr (kKeep == MORPH_FFN_KEEP_FULL) {
    const float* p = static_cast<const float*>(buffer) + at + 4 * fh;
#pragma unroll
    for (int q = 0; q < 4; ++q) k.v[q] = *reinterpret_cast<const f32x4*>(p + 8 * q);
  } else {
    k.codes = *reinterpret_cast<const u32x4*>(static_cast<const uint8_t*>(buffer) + at + 16 * fh);
    k.exponent = exponents[at / MORPH_ACT_GROUP];
  }
}
template <int kKeep>
__device__ __forceinline__ void kept_values(const KeptBlock<kKeep>& k, float (&x)[16]) {
  if constexpr (kKeep == MORPH_FFN_KEEP_FULL) {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = k.v[r >> 2][r & 3];
  } else {
    uint32_t w[4] = {k.codes[0], k.codes[2], k.codes[1], k.codes[3]};
    swap_halves(w[0], w[2]);
    swap_halves(w[1], w[3]);
    const float scale = act_scale((int)k.exponent);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float v[4];
      act_decode4(w[q], scale, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * q + e] = v[e];
    }
  }
}

// ---- the tile -------------------------------------------------------------------

// kPCols, kQCols: how P and Q are stored; kTwo: two segments of K; kKeep: what the gate keeps.
template <int TM, int TN, typename T, bool kPCols, bool kQCols, bool kTwo, FfnEpilogue kE, int kKeep>
__global__ __launch_bounds__(kFfnThreads, (FfnTile<TM, TN>::kPerCu)) void ffn_tile_kernel(const FfnTileArgs g) {
  using C = FfnTile<TM, TN>;
  constexpr int BK = C::kDepth, kSlots = C::kSlots, kSlot = C::kSlot, kBi = C::kBi, kBj = C::kBj;
  constexpr int kLoadsP = TM / 32, kLoadsQ = TN / 32;  // load instructions per wave and slot
  constexpr bool kDual = kE == FfnEpilogue::kGate;
  static_assert(!(kDual && (kPCols || kQCols || kTwo)) && !(kPCols && kTwo), "forms in use");
  __shared__ __attribute__((aligned(16))) uint16_t smem[C::kSmem];

  // The dispatcher hands workgroup i to XCD i % 8; each XCD runs a contiguous range of tiles,
  // numbered in groups of kGroupM tile rows, so that those it runs at a time share panels.
  constexpr int kGroupM = 4;
  const int per_xcd = (int)gridDim.x / 8;
  int t = (int)(blockIdx.x % 8) * per_xcd + (int)blockIdx.x / 8;
  if (t >= g.total) return;
  int which = 0;
  if (g.count > 1 && t >= g.p[1].first) which = 1;
  if (g.count > 2 && t >= g.p[2].first) which = 2;
  const FfnTileProblem& o = g.p[which];
  t -= o.first;
  int tr, tc;
  {
    const int per_group = kGroupM * o.tiles_n, group = t / per_group, within = t - group * per_group;
    const int rows = min(kGroupM, o.tiles_m - group * kGroupM);
    tc = within / rows;
    tr = group * kGroupM + within % rows;
  }
  constexpr int kCols = kDual ? TN / 2 : TN;  // output columns of a tile
  const int row0 = tr * TM, col0 = tc * kCols;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto uniform = [](const uint16_t* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const uint16_t*>(lo | (hi << 32));
  };
  const int K = __builtin_amdgcn_readfirstlane(g.K);
  const int KS = (K + BK - 1) / BK;         // stages of a segment, >= 1
  const int KT = kTwo ? 2 * KS : KS;        // of the product
  constexpr bool kParts = TM <= 128 && kE == FfnEpilogue::kStore;
  const int part = kParts ? (int)blockIdx.y : 0;
  const int first = kParts ? part * KT / g.splits : 0;  // the part's first stage, and how many
  const int count = kParts ? (part + 1) * KT / g.splits - first : KT;
  const int rest = K - (KS - 1) * BK;       // K in a segment's last stage, 1 .. 64

  // One operand's tile: its base, and the descriptor's limits.  "rows": offsets of rows past
  // the end are past ((rows - 1) ld + K) whatever stage the base has advanced to.  "cols": what
  // follows the last stage's base, and a stage more of the ones before it (a tile wider than
  // the matrix reads on into later rows, which end there).  Offsets stay under 2^31 (the
  // host's limit on ld).
  struct Side {
    const uint16_t* base;
    int64_t step;          // elements per stage
    uint32_t limit, last;  // bytes, before the last stage and in it
  };
  constexpr int64_t kMost = 0x7FFFFFFF;
  auto side = [&](const uint16_t* p, int64_t ld, bool cols, int at, int rows, int width) {
    Side s;
    int64_t limit;
    if (cols) {
      s.base = uniform(p + at);
      s.step = BK * ld;
      limit = ((rest - 1) * ld + (width - at)) * 2;
    } else {
      s.base = uniform(p + (int64_t)at * ld);
      s.step = BK;
      limit = ((int64_t)(rows - at - 1) * ld + (K + 7) / 8 * 8) * 2;
    }
    auto clamp = [](int64_t x) {
      return (uint32_t)__builtin_amdgcn_readfirstlane((int)(x < 0 ? 0 : x < kMost ? x : kMost));
    };
    s.last = clamp(limit);
    s.limit = cols ? clamp(limit + 2 * s.step) : s.last;
    return s;
  };
  const Side P0 = side(o.P[0], o.ldp[0], kPCols, row0, o.M, (o.M + 7) / 8 * 8);
  const Side Q0 = side(o.Q[0], o.ldq[0], kQCols, col0, o.N, (o.N + 7) / 8 * 8);
  Side P1 = P0, Q1 = Q0;
  if constexpr (kTwo) P1 = side(o.P[1], o.ldp[1], false, row0, o.M, 0);
  if constexpr (kTwo || kDual) Q1 = side(o.Q[1], o.ldq[1], kQCols, col0, o.N, (o.N + 7) / 8 * 8);

  // Loads.  "rows": wave w loads a quarter of a slot's rows, 8 per instruction; lane l: row l / 8,
  // LDS chunk l % 8, which holds the global chunk (l % 8) ^ swz(row).  "cols": 512 / width of the
  // stage's 64 rows per instruction.  kGate: the LDS rows of Q alternate in blocks of 32 between
  // gate and up, so that a wave's blocks 2j and 2j + 1 are the g and the u of the same
  // columns (at 64: waves 0 and 2 hold the g, 1 and 3 the u).
  const int lrow = lane >> 3, lslot = lane & 7;
  auto swz = [](int r) { return (r ^ (r >> 3)) & 7; };
  // the 4 rows that a transposing read touches land on distinct banks (two rows fill them at 64)
  auto swz_cols = [](int r, int width) { return width == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); };
  auto is_up = [&](int j) { return TN == 256 ? j >= 4 : TN == 128 ? (wave & 1) != 0 : wave >= 2; };  // kGate
  uint32_t offp[kLoadsP], offq[kLoadsQ];
  uint32_t behindp = 0, behindq = 0;  // bit j: load j's chunk of a "rows" operand is past K in the last stage
  auto offset = [&](int j, int width, bool cols, int64_t ld, uint32_t& behind, int tensor_row) {
    if (cols) {
      const int rk = wave * 16 + j * (512 / width) + lane / (width / 8);
      return (uint32_t)rk * (uint32_t)ld * 2u + (uint32_t)((lane % (width / 8)) ^ swz_cols(rk, width)) * 16u;
    }
    const int r = wave * (width / 4) + j * 8 + lrow;
    const uint32_t c = (uint32_t)(lslot ^ swz(r));
    if ((int)c * 8 >= rest) behind |= 1u << j;
    return (uint32_t)(tensor_row >= 0 ? tensor_row : r) * (uint32_t)ld * 2u + c * 16u;
  };
#pragma unroll
  for (int j = 0; j < kLoadsP; ++j) offp[j] = offset(j, TM, kPCols, o.ldp[0], behindp, -1);
#pragma unroll
  for (int j = 0; j < kLoadsQ; ++j) {
    if constexpr (kDual) {
      const int rt = TN == 256   ? wave * 32 + (j & 3) * 8 + lrow
                     : TN == 128 ? (wave >> 1) * 32 + j * 8 + lrow
                                 : (wave & 1) * 16 + j * 8 + lrow;
      offq[j] = offset(j, TN, false, is_up(j) ? o.ldq[1] : o.ldq[0], behindq, rt);
    } else {
      offq[j] = offset(j, TN, kQCols, o.ldq[0], behindq, -1);
    }
  }
  // With a "cols" operand the load is inline assembly: the compiler then adds no waits of its
  // own before the transposing reads.  Completion is managed by the vmcnt waits below.
  auto issue_load = [&](bool q, int slot, int at, int j) {
    const int stage = first + at;
    const bool second = kTwo && stage >= KS;
    const int s = second ? stage - KS : stage;
    const bool last = s == KS - 1;
    Side side = q ? (second ? Q1 : Q0) : (second ? P1 : P0);
    if constexpr (kDual) {
      if (q && is_up(j)) side = Q1;
    }
    const bool cols = q ? kQCols : kPCols;
    const int width = q ? TN : TM;
    const uint16_t* base = side.base + (int64_t)s * side.step;
    const uint32_t limit = cols && last ? side.last : side.limit;
    const uint16_t* dst = smem + slot * kSlot +
                          (cols ? (wave * 16 + j * (512 / width)) * width : (wave * (width / 4) + j * 8) * BK);
    uint32_t off = q ? offq[q ? j : 0] : offp[j];
    if (!cols) off |= ((q ? behindq : behindp) << (31 - j)) & (last ? 0x80000000u : 0u);
    if constexpr (kPCols || kQCols || TM == 64) {
      const uint64_t addr = reinterpret_cast<uint64_t>(uniform(base));
      const u32x4 rsrc = u32x4{(uint32_t)addr, (uint32_t)(addr >> 32) & 0xFFFFu,
                               (uint32_t)__builtin_amdgcn_readfirstlane((int)limit), 0x00020000u};
      const uint32_t m0 = (uint32_t)reinterpret_cast<uintptr_t>(
          (__attribute__((address_space(3))) const uint16_t*)dst);
      // the s_nop is the wait state between a write of M0 and an LDS load
      asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
                   :
                   : "v"(off), "s"(rsrc), "{m0}"(m0)
                   : "memory");
    } else {
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint16_t*>(base), (short)0, (int)limit, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)dst, 16, off, 0, 0, 0);
    }
  };

  const int wr = (wave >> 1) * (TM / 2), wc = (wave & 1) * (TN / 2);
  const int fr = lane & 31, fh = lane >> 5;
  f32x16 acc[kBi][kBj];
#pragma unroll
  for (int i = 0; i < kBi; ++i)
#pragma unroll
    for (int j = 0; j < kBj; ++j) acc[i][j] = f32x16{};

  auto frag = [&](const uint16_t* sub, int R, int c) {
    return *reinterpret_cast<const u32x4*>(sub + R * BK + ((c ^ swz(R)) * 8));
  };
  // Half h of a "cols" operand's fragment of rows n0 .. n0 + 31 at depth kk: in each group of 16
  // lanes the transposing read gives lane j, slot e, element j % 4 of source lane 4 e + j / 4.
  auto frag_cols = [&](const uint16_t* sub, int width, int n0, int kk, int h) {
    const int j = lane & 15;
    const int row = kk * 16 + 8 * (lane >> 5) + 4 * h + (j >> 2);
    const int col = n0 + 16 * ((lane >> 4) & 1) + 4 * (j & 3);
    const uint16_t* at = sub + row * width + ((((col >> 3) ^ swz_cols(row, width)) << 3) | (col & 7));
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (lds_bf16x4*)(__attribute__((address_space(3))) uint16_t*)at));  // used as a whole only
  };
  auto lds_barrier = []() { asm volatile("s_barrier" ::: "memory"); };
  struct Frags {
    u32x4 a[kBi], q[kBj];
  };
  constexpr int kMfmas = kBi * kBj;  // per sub-step of 16 k
  auto mfma = [&](int n, const Frags& f) {
    const int i = n / kBj, j = n % kBj;
    acc[i][j] = mfma32<T>(f.q[j], f.a[i], acc[i][j]);
  };
  constexpr int kPParts = kPCols ? 2 : 1, kQParts = kQCols ? 2 : 1;
  constexpr int kReads = kBi * kPParts + kBj * kQParts;
  // Read n of a sub-step's fragments: P's and Q's in turn, then what is left of P's.
  auto read = [&](int n, Frags& f, int pslot, int qslot, int kk) {
    constexpr int kPair = kPParts + kQParts;
    const bool paired = n < kBj * kPair;
    const int m = paired ? n % kPair : (n - kBj * kPair) % kPParts;
    const int i = paired ? n / kPair : kBj + (n - kBj * kPair) / kPParts;
    const bool q = paired && m >= kPParts;
    const int h = q ? m - kPParts : m;
    const uint16_t* sub = smem + (q ? qslot : pslot) * kSlot;
    const int at = (q ? wc : wr) + i * 32;
    u32x4& to = q ? f.q[q ? i : 0] : f.a[i];
    if (q ? kQCols : kPCols) {
      const u32x2 half = frag_cols(sub, q ? TN : TM, at, kk, h);
      if (h == 0) to.x = half.x, to.y = half.y;
      else to.z = half.x, to.w = half.y;
    } else {
      to = frag(sub, at + fr, kk * 2 + fh);
    }
  };

  // kGateGrad: what was kept of the first blocks is on its way under the last stage's MFMAs, and
  // kAhead blocks ahead of its use from then on (4096 rows of 3072 x 6144: 278 us, 296 with a wait per block).
  constexpr int kAhead = kE != FfnEpilogue::kGateGrad || TM == 64 ? 1 : kKeep == MORPH_FFN_KEEP_FULL ? 3 : 4;
  [[maybe_unused]] KeptBlock<kKeep> kg[kAhead], ku[kAhead] = {};
  auto load_block = [&](int n) {
    if constexpr (kE == FfnEpilogue::kGateGrad) {
      const int row = row0 + wr + 32 * (n / kBj) + fr, block = col0 + wc + 32 * (n % kBj);
      if (block >= o.ldc) return;
      const int64_t at = (int64_t)min(row, o.M - 1) * o.ldc + block;
      load_kept<kKeep>(kg[n % kAhead], g.g, g.g_exponents, at, fh);
      load_kept<kKeep>(ku[n % kAhead], g.u, g.u_exponents, at, fh);
    }
  };
  auto load_ahead = [&]() {
    if constexpr (kE == FfnEpilogue::kGateGrad) {
#pragma unroll
      for (int n = 0; n < kAhead; ++n) load_block(n);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if constexpr (TM == 64) {
    // A ring of whole stages, and two register sets that hold all fragments of a stage each: step t
    // waits until stage t + 1 has landed, the barrier publishes it and frees stage t's slots, and
    // the reads of t + 1 and the loads of t + 3 run under stage t's MFMAs.
    constexpr int kRing = kSlots / 2, kStageLoads = kLoadsP + kLoadsQ;
    struct Stage {
      Frags f[4];
    };
    auto load_stage = [&](int slot, int stage) {
#pragma unroll
      for (int j = 0; j < kLoadsP; ++j) issue_load(false, 2 * slot, stage, j);
#pragma unroll
      for (int j = 0; j < kLoadsQ; ++j) issue_load(true, 2 * slot + 1, stage, j);
    };
    auto read_stage = [&](Stage& st, int slot) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int n = 0; n < kReads; ++n) read(n, st.f[kk], 2 * slot, 2 * slot + 1, kk);
    };
    // this wave's loads of all but the youngest `pending` stages have landed
    static_assert(kRing <= 3 && 2 * kStageLoads < 16, "the counts of wait_pending");
    auto wait_pending = [&](int pending) {
      if (pending <= 0) __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      else if (pending == 1) __builtin_amdgcn_s_waitcnt(0x0F70 | kStageLoads);
      else __builtin_amdgcn_s_waitcnt(0x0F70 | (2 * kStageLoads));
    };
    Stage s0, s1;
    int slot = 0;  // of stage t
    auto step = [&](int t, const Stage& cur, Stage& nxt) {
      const int nslot = slot + 1 == kRing ? 0 : slot + 1;
      if (t + 1 < count) {
        wait_pending(min(kRing - 1, count - 1 - t) - 1);
        lds_barrier();
        read_stage(nxt, nslot);
        if (t + kRing < count) load_stage(slot, t + kRing);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) mfma(0, cur.f[kk]);
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): next fragments in registers
      slot = nslot;
    };
#pragma unroll
    for (int k = 0; k < kRing; ++k)
      if (k < count) load_stage(k, k);
    wait_pending(min(kRing, count) - 1);
    lds_barrier();
    read_stage(s0, 0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    for (int t = 0; t + 1 < count; t += 2) {
      step(t, s0, s1);
      step(t + 1, s1, s0);
    }
    load_ahead();
    if (count & 1) step(count - 1, s0, s1);
  } else {
    Frags f0, f1;
    constexpr int kHalfP = kLoadsP / 2, kHalfQ = kLoadsQ / 2;
    constexpr int kPre = TM == 256 ? 2 : 1;  // MFMAs of the last sub-step before the barrier
    // Behind MFMA n of a sub-step whose reads start after MFMA `first`: one or two reads at a
    // time, at 128 x 128 half of them behind each of two MFMAs.
    auto reads_behind = [&](int n, int first, Frags& nxt, int rp, int rq, int kk) {
      constexpr int kEach = TM == 256 ? (kReads + kMfmas - kPre - 1) / (kMfmas - kPre) : kReads / 2;
#pragma unroll
      for (int k = 0; k < kEach; ++k)
        if (n >= first && (n - first) * kEach + k < kReads) read((n - first) * kEach + k, nxt, rp, rq, kk);
    };
    // Loads j0 on, half a slot's: one behind every other MFMA (256 x 256), every one (256 x 128),
    // or all at once.
    auto loads_behind = [&](int n, int first, bool lq, int ls_, int lstage, bool upper) {
      const int half = lq ? kHalfQ : kHalfP, j0 = upper ? half : 0;
      if constexpr (TM == 256) {
        constexpr int kStep = TN == 256 ? 2 : 1;
        const int l = (n - first - kStep) / kStep;
        if (n >= first + kStep && (n - first) % kStep == 0 && l < half) issue_load(lq, ls_, lstage, j0 + l);
      } else if (n == first) {
#pragma unroll
        for (int j = 0; j < half; ++j) issue_load(lq, ls_, lstage, j0 + j);
      }
    };
    auto substep = [&](const Frags& cur, Frags& nxt, int rp, int rq, int kk, auto load, bool lq, int ls_,
                       int lstage, bool upper) {
#pragma unroll
      for (int n = 0; n < kMfmas; ++n) {
        mfma(n, cur);
        __builtin_amdgcn_sched_barrier(0);
        reads_behind(n, 0, nxt, rp, rq, kk);
        if constexpr (decltype(load)::value) loads_behind(n, 0, lq, ls_, lstage, upper);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): next fragments in registers
    };
    // Step t computes stage t in four sub-steps, whose MFMAs run while the next sub-step's fragments
    // are read.  kind: 0 with stages t + 1 and t + 2 to come, 1 the last but one, 2 the last.
    auto step = [&](int t, int ps, auto kind) {
      constexpr bool kNext = decltype(kind)::value < 2, kNext2 = decltype(kind)::value == 0;
      const int qs = ps + 1 == kSlots ? 0 : ps + 1;
      const int ps1 = qs + 1 == kSlots ? 0 : qs + 1;
      const int qs1 = ps1 + 1 == kSlots ? 0 : ps1 + 1;
      const int ps2 = qs1 + 1 == kSlots ? 0 : qs1 + 1;
      const std::bool_constant<kNext> l1;
      const std::bool_constant<kNext2> l2;
      substep(f0, f1, ps, qs, 1, l1, true, qs1, t + 1, true);    // Q of t + 1, second half
      substep(f1, f0, ps, qs, 2, l2, false, ps2, t + 2, false);  // P of t + 2, first half
      substep(f0, f1, ps, qs, 3, l2, false, ps2, t + 2, true);   // P of t + 2, second half
#pragma unroll
      for (int n = 0; n < kPre; ++n) mfma(n, f1);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kNext) {
        // all but P of t + 2 landed for this wave; the barrier publishes stage t + 1 and frees
        // stage t's slots (every wave holds its last fragments)
        __builtin_amdgcn_s_waitcnt(0x0F70 | (kNext2 ? kLoadsP : 0));
        lds_barrier();
      }
#pragma unroll
      for (int n = kPre; n < kMfmas; ++n) {
        mfma(n, f1);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kNext) {
          reads_behind(n, kPre, f0, ps1, qs1, 0);
          // Q of t + 2 into the freed P slot of t, first half
          if constexpr (kNext2) loads_behind(n, TN == 256 ? 4 : kPre, true, ps, t + 2, false);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (kNext) __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    };
#pragma unroll
    for (int j = 0; j < kLoadsP; ++j) issue_load(false, 0, 0, j);
#pragma unroll
    for (int j = 0; j < kLoadsQ; ++j) issue_load(true, 1, 0, j);
    if (count > 1) {
#pragma unroll
      for (int j = 0; j < kLoadsP; ++j) issue_load(false, 2, 1, j);
#pragma unroll
      for (int j = 0; j < kHalfQ; ++j) issue_load(true, 3, 1, j);
      __builtin_amdgcn_s_waitcnt(0x0F70 | (kLoadsP + kHalfQ));  // P and Q of stage 0 landed for this wave
    } else {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    }
    lds_barrier();
#pragma unroll
    for (int n = 0; n < kReads; ++n) read(n, f0, 0, 1, 0);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    int ps = 0;
    auto advance = [&]() { ps = ps + 2 >= kSlots ? ps + 2 - kSlots : ps + 2; };
    for (int t = 0; t + 2 < count; ++t) {
      step(t, ps, std::integral_constant<int, 0>{});
      advance();
    }
    if (count > 1) {
      step(count - 2, ps, std::integral_constant<int, 1>{});
      advance();
    }
    load_ahead();
    step(count - 1, ps, std::integral_constant<int, 2>{});
  }

  // ---- epilogue: straight from the registers ------------------------------------
  const int M = o.M, N = o.N;
  const int64_t ldc = o.ldc;
  // h, and g and u as they are kept, of a 32 x 32 block
  [[maybe_unused]] auto gate_block = [&](int row, int block, const float (&gv)[16], const float (&uv)[16],
                                         const float (&h)[16]) {
    const bool inside = row < M;
    const int64_t at = (int64_t)row * ldc + block;
    u32x4 lo, hi;
    row_words<T>(h, lo, hi);
    if (inside) {
      *reinterpret_cast<u32x4*>(o.C + at + 16 * fh) = lo;
      *reinterpret_cast<u32x4*>(o.C + at + 16 * fh + 8) = hi;
    }
    keep_block<kKeep>(gv, g.g, g.g_exponents, at, fh, inside);
    keep_block<kKeep>(uv, g.u, g.u_exponents, at, fh, inside);
  };
  if constexpr (kE == FfnEpilogue::kStore) {
#pragma unroll
    for (int i = 0; i < kBi; ++i) {
      const int row = row0 + wr + 32 * i + fr;
#pragma unroll
      for (int j = 0; j < kBj; ++j) {
        const int block = col0 + wc + 32 * j;
        float x[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = acc[i][j][r];
        if (kParts && g.splits > 1) {
          if (row >= M) continue;
          float* at = g.parts + ((int64_t)part * M + row) * (o.tiles_n * TN) + block + 4 * fh;
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(at + 8 * q) = f32x4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
          continue;
        }
        u32x4 w[2];
        row_words<T>(x, w[0], w[1]);
        const int col = block + 16 * fh;
        uint16_t* at = o.C + (int64_t)row * ldc + col;
        if (row >= M) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k) store_eight(at + 8 * k, w[k], N - col - 8 * k, o.vector != 0);
      }
    }
  } else if constexpr (kE == FfnEpilogue::kGate && TM == 64) {
    // waves 0 and 2 hold g of 32 rows each, 1 and 3 the u of the same: they meet through LDS
    __syncthreads();  // every wave's fragment reads are done
    f32x4* meet = reinterpret_cast<f32x4*>(smem) + (wave >> 1) * 256 + lane;
    if (wave & 1) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        meet[64 * q] = f32x4{acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]};
    }
    __syncthreads();
    if (wave & 1) return;
    const int row = row0 + wr + fr;
    float gv[16], uv[16], h[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      gv[r] = acc[0][0][r], uv[r] = meet[64 * (r >> 2)][r & 3];
      h[r] = ffn_gate(gv[r], uv[r]);
    }
    gate_block(row, col0, gv, uv, h);
  } else if constexpr (kE == FfnEpilogue::kGate) {
#pragma unroll
    for (int i = 0; i < kBi; ++i) {
      const int row = row0 + wr + 32 * i + fr;
#pragma unroll
      for (int j = 0; j < kBj / 2; ++j) {
        const int block = col0 + (wc + 64 * j) / 2;
        if (block >= ldc) continue;  // rows of the buffers are whole groups
        float gv[16], uv[16], h[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          gv[r] = acc[i][2 * j][r], uv[r] = acc[i][2 * j + 1][r];
          h[r] = ffn_gate(gv[r], uv[r]);
        }
        gate_block(row, block, gv, uv, h);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kBi; ++i) {
      const int row = row0 + wr + 32 * i + fr;
      const bool inside = row < M;
#pragma unroll
      for (int j = 0; j < kBj; ++j) {
        const int block = col0 + wc + 32 * j;
        const int64_t at = (int64_t)row * ldc + block;
        float gv[16], uv[16], h[16];
        kept_values<kKeep>(kg[(i * kBj + j) % kAhead], gv);
        kept_values<kKeep>(ku[(i * kBj + j) % kAhead], uv);
        if (i * kBj + j + kAhead < kBi * kBj) load_block(i * kBj + j + kAhead);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const GateGrad d = ffn_gate_grad(acc[i][j][r], gv[r], uv[r]);
          h[r] = d.h, gv[r] = d.dg, uv[r] = d.du;
        }
        if (block + 32 > N) {  // columns behind N are zero in every buffer; the sums there are not
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (block + 8 * (r >> 2) + 4 * fh + (r & 3) >= N) h[r] = gv[r] = uv[r] = 0.0f;
        }
        u32x4 w[6];
        row_words<T>(h, w[0], w[1]);
        row_words<T>(gv, w[2], w[3]);
        row_words<T>(uv, w[4], w[5]);
        if (inside && block < ldc) {  // rows of the buffers are whole groups
          uint16_t* to[3] = {o.C, g.dg, g.du};
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            *reinterpret_cast<u32x4*>(to[k] + at + 16 * fh) = w[2 * k];
            *reinterpret_cast<u32x4*>(to[k] + at + 16 * fh + 8) = w[2 * k + 1];
          }
        }
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------

// The tiles' shapes.
enum FfnShape { kTile256, kTile256x128, kTile128, kTile64, kFfnShapes };
constexpr int kFfnTileM[kFfnShapes] = {256, 256, 128, 64}, kFfnTileN[kFfnShapes] = {256, 128, 128, 64};

// The forms that the block needs, each in a source file of its own kind:
// gate: x gate^T and x up^T -> h and what is kept; rows: h down^T -> y; grad: dy down -> h, dg,
// du; two: dg gate + du up -> dx; weights: dg^T x, du^T x, dy^T h.
__attribute__((visibility("hidden"))) void ffn_tile_gate(FfnShape shape, int dtype, int keep, unsigned grid, hipStream_t s,
                                                         const FfnTileArgs& a);
__attribute__((visibility("hidden"))) void ffn_tile_rows(FfnShape shape, int dtype, unsigned grid, hipStream_t s,
                                                         const FfnTileArgs& a);
__attribute__((visibility("hidden"))) void ffn_tile_grad(FfnShape shape, int dtype, int keep, unsigned grid, hipStream_t s,
                                                         const FfnTileArgs& a);
__attribute__((visibility("hidden"))) void ffn_tile_two(FfnShape shape, int dtype, unsigned grid, hipStream_t s,
                                                        const FfnTileArgs& a);
__attribute__((visibility("hidden"))) void ffn_tile_weights(FfnShape shape, int dtype, unsigned grid, hipStream_t s,
                                                            const FfnTileArgs& a);

template <bool kPCols, bool kQCols, bool kTwo, FfnEpilogue kE, int kKeep>
void launch_ffn_tiles(FfnShape shape, int dtype, unsigned grid, hipStream_t s, const FfnTileArgs& a) {
  const dim3 gd(grid, (unsigned)a.splits), bd(kFfnThreads);
  auto with = [&](auto type) {
    typedef decltype(type) T;
    switch (shape) {
      case kTile256: hipLaunchKernelGGL((ffn_tile_kernel<256, 256, T, kPCols, kQCols, kTwo, kE, kKeep>), gd, bd, 0, s, a); break;
      case kTile256x128: hipLaunchKernelGGL((ffn_tile_kernel<256, 128, T, kPCols, kQCols, kTwo, kE, kKeep>), gd, bd, 0, s, a); break;
      case kTile128: hipLaunchKernelGGL((ffn_tile_kernel<128, 128, T, kPCols, kQCols, kTwo, kE, kKeep>), gd, bd, 0, s, a); break;
      default: hipLaunchKernelGGL((ffn_tile_kernel<64, 64, T, kPCols, kQCols, kTwo, kE, kKeep>), gd, bd, 0, s, a); break;
    }
  };
  if (dtype == MORPH_DTYPE_F16) with(F16{});
  else with(BF16{});
}

}  // namespace morph
