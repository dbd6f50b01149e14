// mlk_ragged_few_64_scored.hip -- the kernels of mlk_ragged_few.h for head_dim up to 64, with score functions and masks.
#include "mlk_ragged_few.h"

namespace mlk {
template mlk_status LaunchFewAt<64, true>(const RaggedParams&, dim3, int32_t, int32_t, hipStream_t);
}  // namespace mlk
