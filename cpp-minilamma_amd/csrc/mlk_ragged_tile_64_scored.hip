// mlk_ragged_tile_64_scored.hip -- the kernels of mlk_ragged_tile.h for head_dim up to 64, with score functions and masks.
#include "mlk_ragged_tile.h"

namespace mlk {
template mlk_status LaunchTileAt<64, true>(const RaggedParams&, dim3, int64_t, int32_t, int32_t, hipStream_t);
}  // namespace mlk
