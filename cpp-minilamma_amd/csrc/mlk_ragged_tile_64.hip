// mlk_ragged_tile_64.hip -- the kernels of mlk_ragged_tile.h for head_dim up to 64.
#include "mlk_ragged_tile.h"

namespace mlk {
template mlk_status LaunchTileAt<64, false>(const RaggedParams&, dim3, int64_t, int32_t, int32_t, hipStream_t);
}  // namespace mlk
