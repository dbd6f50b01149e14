// mlk_ragged_few_128.hip -- the kernels of mlk_ragged_few.h for head_dim 65 to 128.
#include "mlk_ragged_few.h"

namespace mlk {
template mlk_status LaunchFewAt<128, false>(const RaggedParams&, dim3, int32_t, int32_t, hipStream_t);
}  // namespace mlk
