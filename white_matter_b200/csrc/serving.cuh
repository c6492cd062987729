// Shared by the serving operators: element types of a pool on the device, and the launchers behind
// include/wm_b200_serving.h.
#pragma once

#include "common.cuh"
#include "wm_b200_serving.h"

namespace wm {

constexpr int kMaxTreeNodes = 512;      // drafted tokens per tree
constexpr int kMaxSlots = 0x7fffff00;  // of a pool: the kernels step a few rows past the last one in 32 bits

int pool_commit_launch(const wm_pool_commit_args& a, cudaStream_t stream);
int pool_advance_launch(void* lengths, int lengths_is64, const int32_t* index, const int32_t* counts, int batch, int rows, int source_rows, int capacity, cudaStream_t stream);
int pool_dequant_launch(const wm_pool_dequant_args& a, cudaStream_t stream);
int draft_tree_launch(const wm_draft_tree_args& a, cudaStream_t stream);
int pool_attn_launch(const wm_pool_attn_args& a, cudaStream_t stream);
size_t pool_attn_workspace(const wm_pool_attn_args& a);

// the four codes of a word as fp32 numbers, element 0 in the low byte
__device__ __forceinline__ void codes_to_float(uint32_t w, bool is_int8, float* x) {
  if (is_int8) {
    // code + 128 as the low byte of 2^23 + code + 128: exact, and no conversion instruction, of which an SM does 16 a cycle
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(__byte_perm(w ^ 0x80808080u, 0x4b000000u, 0x7540 + i)) - 8388736.f;
  } else {
    uint32_t lo, hi;  // two halves each; every e4m3 number is an fp16 number
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(static_cast<uint16_t>(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(static_cast<uint16_t>(w >> 16)));
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h;}" : "=f"(x[0]), "=f"(x[1]) : "r"(lo));
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h;}" : "=f"(x[2]), "=f"(x[3]) : "r"(hi));
  }
}

}  // namespace wm
