// The tile kernels of head_tile.h for f16 operands.
#include "head_tile.h"

namespace pngpd {
hipError_t launch_tile_f16(int shape, int kind, bool ak, bool bk, const TileArgs& g, hipStream_t s) {
    return launch_tile<f16_t>(shape, kind, ak, bk, g, s);
}
hipError_t launch_pair_f16(const TileArgs& x, const TileArgs& w, hipStream_t s) {
    return launch_pair<f16_t>(x, w, s);
}
}  // namespace pngpd
