// The tile kernels of head_tile.h for float operands.
#include "head_tile.h"

namespace pngpd {
hipError_t launch_tile_f32(int shape, int kind, bool ak, bool bk, const TileArgs& g, bool vec, hipStream_t s) {
    return launch_tile<float>(shape, kind, ak, bk, g, vec, s);
}
}  // namespace pngpd
