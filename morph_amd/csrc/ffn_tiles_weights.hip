// The weight gradients, dg^T x, du^T x and dy^T h (ffn_tiles.h).
#include "ffn_tiles.h"

void morph::ffn_tile_weights(FfnShape shape, int dtype, unsigned grid, hipStream_t s, const FfnTileArgs& a) {
  launch_ffn_tiles<true, true, false, FfnEpilogue::kStore, MORPH_FFN_KEEP_NONE>(shape, dtype, grid, s, a);
}
