// The query side of the backward of structure attention on the tensor cores.
#include "structure_attention_tile.cuh"

namespace y3b {

int attention_query_tiles(int pieces, AttTileArgs& a, int64_t items, cudaStream_t s) {
  return dispatch_attention_tile<kQuerySide>(pieces, a, items, s);
}

}  // namespace y3b
