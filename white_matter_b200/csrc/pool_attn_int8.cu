// Pool attention over int8 pools (see pool_attn_mma.cuh).
#include "pool_attn_mma.cuh"

namespace wm {
namespace pool {
WM_POOL_ATTN_UNIT(WM_INT8, false)
}  // namespace pool
}  // namespace wm
