// Row tiles of MXFP4 x and weights (expert_tile.h).
#include "expert_tile.h"

namespace lf {
namespace expert {

int launch_tiles_mx(const Params& p, int cap, int columns, hipStream_t stream) {
  switch (columns) {
    case 64: return tile::launch<true, true, 1>(p, cap, stream);
    case 128: return tile::launch<true, true, 2>(p, cap, stream);
    case 192: return tile::launch<true, true, 3>(p, cap, stream);
    default: return tile::launch<true, true, 4>(p, cap, stream);
  }
}

}  // namespace expert
}  // namespace lf
