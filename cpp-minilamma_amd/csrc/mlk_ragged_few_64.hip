// mlk_ragged_few_64.hip -- the kernels of mlk_ragged_few.h for head_dim up to 64.
#include "mlk_ragged_few.h"

namespace mlk {
template mlk_status LaunchFewAt<64, false>(const RaggedParams&, dim3, int32_t, int32_t, hipStream_t);
}  // namespace mlk
