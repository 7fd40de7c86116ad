// The gated feed-forward block of few rows (ffn_rows.hip).
#pragma once

#include "ffn.h"

namespace morph {

constexpr int64_t kFewRows = 64;

// h = silu(x gate^T) * (x up^T) (gated: Q0 = gate, Q1 = up) or C = P Q0^T for P [M, K], Q [N, K],
// 1 <= M <= kFewRows, rows at any 2-byte alignment and stride.
__attribute__((visibility("hidden"))) int ffn_few_rows(int dtype, bool gated, const uint16_t* P, int64_t ldp,
                                                       const uint16_t* Q0, int64_t ldq0, const uint16_t* Q1,
                                                       int64_t ldq1, int64_t M, int64_t N, int64_t K, uint16_t* C,
                                                       int64_t ldc, hipStream_t s);

}  // namespace morph
