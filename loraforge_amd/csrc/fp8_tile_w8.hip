// Row tiles of bf16 x and FP8 weights (fp8_tile.h).
#include "fp8_tile.h"

namespace lf {
namespace expert {

int launch_tiles_w8(const Params& p, int cap, int columns, hipStream_t stream) { return tile8::launch<false>(p, cap, columns, stream); }

}  // namespace expert
}  // namespace lf
