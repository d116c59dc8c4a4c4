// Attention over a shared prefix, head_dim 128, bf16 values.
#include "paged_prefix.cuh"

namespace sunshape {
SUNSHAPE_PREFIX_INSTANCES(128, __nv_bfloat16)
}  // namespace sunshape
