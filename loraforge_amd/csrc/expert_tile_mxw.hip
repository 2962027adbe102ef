// Row tiles of bf16 x and MXFP4 weights (expert_tile.h).
#include "expert_tile.h"

namespace lf {
namespace expert {

int launch_tiles_mxw(const Params& p, int cap, int columns, hipStream_t stream) {
  switch (columns) {
    case 64: return tile::launch<false, true, 1>(p, cap, stream);
    case 128: return tile::launch<false, true, 2>(p, cap, stream);
    case 192: return tile::launch<false, true, 3>(p, cap, stream);
    default: return tile::launch<false, true, 4>(p, cap, stream);
  }
}

}  // namespace expert
}  // namespace lf
