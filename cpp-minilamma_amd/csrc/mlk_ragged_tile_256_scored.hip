// mlk_ragged_tile_256_scored.hip -- the kernels of mlk_ragged_tile.h for head_dim 129 to 256, with score functions and masks.
#include "mlk_ragged_tile.h"

namespace mlk {
template mlk_status LaunchTileAt<256, true>(const RaggedParams&, dim3, int64_t, int32_t, int32_t, hipStream_t);
}  // namespace mlk
