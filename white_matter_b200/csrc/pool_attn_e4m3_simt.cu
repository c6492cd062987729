// Pool attention of fp32 queries over e4m3 pools (see pool_attn_simt.cuh).
#include "pool_attn_simt.cuh"

namespace wm {
namespace pool {
WM_POOL_SIMT_UNIT(WM_E4M3)
}  // namespace pool
}  // namespace wm
