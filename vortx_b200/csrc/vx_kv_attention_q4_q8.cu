// The attention kernel for keys in Q4_0 and values in Q8_0.
#include <type_traits>

#include "vx_kv_attention.cuh"

namespace vx {
VX_ATTN_INSTANCE(true, false)
}  // namespace vx
