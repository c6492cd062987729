// Pool attention over int8 pools, many rows per KV head (see pool_attn_shared.cuh).
#include "pool_attn_shared.cuh"

namespace wm {
namespace pool {
WM_POOL_SHARED_UNIT(WM_INT8)
}  // namespace pool
}  // namespace wm
