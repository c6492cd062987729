// Pool attention of fp32 queries over fp32 pools (see pool_attn_simt.cuh).
#include "pool_attn_simt.cuh"

namespace wm {
namespace pool {
WM_POOL_SIMT_UNIT(WM_F32)
}  // namespace pool
}  // namespace wm
