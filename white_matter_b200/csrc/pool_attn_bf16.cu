// Pool attention over bf16 pools (see pool_attn_mma.cuh).
#include "pool_attn_mma.cuh"

namespace wm {
namespace pool {

void launch_mma_bf16(const wm_pool_attn_args& a, const Plan& plan, int shares, cudaStream_t stream) {
  launch_mma_storage<WM_BF16>(a, plan, shares, stream);
}

}  // namespace pool
}  // namespace wm
