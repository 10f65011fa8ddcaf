// The tile kernels of head_tile.h for float operands.
#include "head_tile.h"

namespace pngpd {
hipError_t launch_tile_f32(int shape, int kind, bool ak, bool bk, const TileArgs& g, hipStream_t s) {
    return launch_tile<float>(shape, kind, ak, bk, g, s);
}
hipError_t launch_pair_f32(const TileArgs& x, const TileArgs& w, hipStream_t s) {
    return launch_pair<float>(x, w, s);
}
}  // namespace pngpd
