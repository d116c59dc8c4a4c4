// Attention over a shared prefix, head_dim 64, bf16 values.
#include "paged_prefix.cuh"

namespace sunshape {
SUNSHAPE_PREFIX_INSTANCES(64, __nv_bfloat16)
}  // namespace sunshape
