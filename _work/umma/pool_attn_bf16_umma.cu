// Pool attention over bf16 pools on tcgen05 (see pool_attn_umma.cuh).
#include <atomic>

#include "pool_attn_umma.cuh"

namespace wm {
namespace pool {
WM_POOL_UMMA_UNIT(WM_BF16)
}  // namespace pool
}  // namespace wm
