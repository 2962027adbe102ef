// Row tiles of bf16 x and weights (expert_tile.h).
#include "expert_tile.h"

namespace lf {
namespace expert {

int launch_tiles_bf16(const Params& p, int cap, int columns, hipStream_t stream) {
  switch (columns) {
    case 64: return tile::launch<false, false, 1>(p, cap, stream);
    case 128: return tile::launch<false, false, 2>(p, cap, stream);
    case 192: return tile::launch<false, false, 3>(p, cap, stream);
    default: return tile::launch<false, false, 4>(p, cap, stream);
  }
}

}  // namespace expert
}  // namespace lf
