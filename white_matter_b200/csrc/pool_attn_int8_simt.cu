// Pool attention of fp32 queries over int8 pools (see pool_attn_simt.cuh).
#include "pool_attn_simt.cuh"

namespace wm {
namespace pool {
WM_POOL_SIMT_UNIT(WM_INT8)
}  // namespace pool
}  // namespace wm
