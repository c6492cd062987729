// Pool attention over bf16 pools, many rows per KV head (see pool_attn_shared.cuh).
#include "pool_attn_shared.cuh"

namespace wm {
namespace pool {
WM_POOL_SHARED_UNIT(WM_BF16)
}  // namespace pool
}  // namespace wm
