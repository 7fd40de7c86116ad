// The forward's first product: x gate^T and x up^T with the gate (ffn_tiles.h).
#include "ffn_tiles.h"

void morph::ffn_tile_gate(FfnShape shape, int dtype, int keep, unsigned grid, hipStream_t s, const FfnTileArgs& a) {
  if (keep == MORPH_FFN_KEEP_FULL)
    launch_ffn_tiles<false, false, false, FfnEpilogue::kGate, MORPH_FFN_KEEP_FULL>(shape, dtype, grid, s, a);
  else if (keep == MORPH_FFN_KEEP_ACT8)
    launch_ffn_tiles<false, false, false, FfnEpilogue::kGate, MORPH_FFN_KEEP_ACT8>(shape, dtype, grid, s, a);
  else
    launch_ffn_tiles<false, false, false, FfnEpilogue::kGate, MORPH_FFN_KEEP_NONE>(shape, dtype, grid, s, a);
}
