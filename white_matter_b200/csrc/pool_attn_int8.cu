// Pool attention over pools held in int8 (see pool_attn_mma.cuh).
#include "pool_attn_mma.cuh"

namespace wm {
namespace pool {

void launch_mma_int8(const wm_pool_attn_args& a, const Plan& plan, int shares, cudaStream_t stream) {
  launch_mma_storage<WM_INT8>(a, plan, shares, stream);
}

}  // namespace pool
}  // namespace wm
