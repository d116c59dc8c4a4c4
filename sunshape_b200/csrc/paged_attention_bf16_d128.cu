// Paged attention, head_dim 128, bf16 values.
#include "paged_attention_kernel.cuh"

namespace sunshape {
SUNSHAPE_PAGED_INSTANCES(128, __nv_bfloat16)
}  // namespace sunshape
