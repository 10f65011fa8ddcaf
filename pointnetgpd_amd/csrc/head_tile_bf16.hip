// The tile kernels of head_tile.h for bf16 operands.
#include "head_tile.h"

namespace pngpd {
hipError_t launch_tile_bf16(int shape, int kind, bool ak, bool bk, const TileArgs& g, hipStream_t s) {
    return launch_tile<bf16_t>(shape, kind, ak, bk, g, s);
}
hipError_t launch_pair_bf16(const TileArgs& x, const TileArgs& w, hipStream_t s) {
    return launch_pair<bf16_t>(x, w, s);
}
}  // namespace pngpd
