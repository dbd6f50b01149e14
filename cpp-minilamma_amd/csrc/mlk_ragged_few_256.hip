// mlk_ragged_few_256.hip -- the kernels of mlk_ragged_few.h for head_dim 129 to 256.
#include "mlk_ragged_few.h"

namespace mlk {
template mlk_status LaunchFewAt<256, false>(const RaggedParams&, dim3, int32_t, int32_t, hipStream_t);
}  // namespace mlk
