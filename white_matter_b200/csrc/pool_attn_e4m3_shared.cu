// Pool attention over e4m3 pools, many rows per KV head (see pool_attn_shared.cuh).
#include "pool_attn_shared.cuh"

namespace wm {
namespace pool {
WM_POOL_SHARED_UNIT(WM_E4M3)
}  // namespace pool
}  // namespace wm
