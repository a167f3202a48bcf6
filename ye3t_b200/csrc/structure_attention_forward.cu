// The forward of structure attention on the tensor cores.
#include "structure_attention_tile.cuh"

namespace y3b {

int attention_forward_tiles(int pieces, AttTileArgs& a, int64_t items, cudaStream_t s) {
  return dispatch_attention_tile<kForward>(pieces, a, items, s);
}

}  // namespace y3b
