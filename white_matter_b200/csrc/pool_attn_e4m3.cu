// Pool attention over pools held in e4m3 (see pool_attn_mma.cuh).
#include "pool_attn_mma.cuh"

namespace wm {
namespace pool {

void launch_mma_e4m3(const wm_pool_attn_args& a, const Plan& plan, int shares, cudaStream_t stream) {
  launch_mma_storage<WM_E4M3>(a, plan, shares, stream);
}

}  // namespace pool
}  // namespace wm
