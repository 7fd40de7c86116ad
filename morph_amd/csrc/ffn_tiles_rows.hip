// The forward's second product, h down^T, and the backward's dx = dg gate + du up (ffn_tiles.h).
#include "ffn_tiles.h"

void morph::ffn_tile_rows(FfnShape shape, int dtype, unsigned grid, hipStream_t s, const FfnTileArgs& a) {
  launch_ffn_tiles<false, false, false, FfnEpilogue::kStore, MORPH_FFN_KEEP_NONE>(shape, dtype, grid, s, a);
}

void morph::ffn_tile_two(FfnShape shape, int dtype, unsigned grid, hipStream_t s, const FfnTileArgs& a) {
  launch_ffn_tiles<false, true, true, FfnEpilogue::kStore, MORPH_FFN_KEEP_NONE>(shape, dtype, grid, s, a);
}
