// mlk_ragged_tile_128.hip -- the kernels of mlk_ragged_tile.h for head_dim 65 to 128.
#include "mlk_ragged_tile.h"

namespace mlk {
template mlk_status LaunchTileAt<128, false>(const RaggedParams&, dim3, int64_t, int32_t, int32_t, hipStream_t);
}  // namespace mlk
