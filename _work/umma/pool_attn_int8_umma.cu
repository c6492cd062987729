// Pool attention over int8 pools on tcgen05 (see pool_attn_umma.cuh).
#include <atomic>

#include "pool_attn_umma.cuh"

namespace wm {
namespace pool {
WM_POOL_UMMA_UNIT(WM_INT8)
}  // namespace pool
}  // namespace wm
