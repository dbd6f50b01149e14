// mlk_ragged_tile_256.hip -- the kernels of mlk_ragged_tile.h for head_dim 129 to 256.
#include "mlk_ragged_tile.h"

namespace mlk {
template mlk_status LaunchTileAt<256, false>(const RaggedParams&, dim3, int64_t, int32_t, int32_t, hipStream_t);
}  // namespace mlk
