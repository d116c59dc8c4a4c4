// Paged attention, head_dim 64, bf16 values.
#include "paged_attention_kernel.cuh"

namespace sunshape {
SUNSHAPE_PAGED_INSTANCES(64, __nv_bfloat16)
}  // namespace sunshape
