// Pool attention over e4m3 pools with drafted tokens (see pool_attn_mma.cuh).
#include "pool_attn_mma.cuh"

namespace wm {
namespace pool {
WM_POOL_ATTN_UNIT(WM_E4M3, true)
}  // namespace pool
}  // namespace wm
