// Pool attention over bf16 pools with drafted tokens (see pool_attn_mma.cuh).
#include "pool_attn_mma.cuh"

namespace wm {
namespace pool {
WM_POOL_ATTN_UNIT(WM_BF16, true)
}  // namespace pool
}  // namespace wm
