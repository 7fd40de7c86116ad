// The backward's first product: dy down with the gate's gradient (ffn_tiles.h).
#include "ffn_tiles.h"

void morph::ffn_tile_grad(FfnShape shape, int dtype, int keep, unsigned grid, hipStream_t s, const FfnTileArgs& a) {
  if (keep == MORPH_FFN_KEEP_FULL)
    launch_ffn_tiles<false, true, false, FfnEpilogue::kGateGrad, MORPH_FFN_KEEP_FULL>(shape, dtype, grid, s, a);
  else
    launch_ffn_tiles<false, true, false, FfnEpilogue::kGateGrad, MORPH_FFN_KEEP_ACT8>(shape, dtype, grid, s, a);
}
