// Attention over a shared prefix, head_dim 128, f16 values.
#include "paged_prefix.cuh"

namespace sunshape {
SUNSHAPE_PREFIX_INSTANCES(128, __half)
}  // namespace sunshape
