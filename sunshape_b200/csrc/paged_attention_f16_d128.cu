// Paged attention, head_dim 128, f16 values.
#include "paged_attention_kernel.cuh"

namespace sunshape {
SUNSHAPE_PAGED_INSTANCES(128, __half)
}  // namespace sunshape
