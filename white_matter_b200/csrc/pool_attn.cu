// Attention of queries that stand behind the committed tokens of a pool -- one token per sequence, a few new ones, or a
// tree of drafted tokens -- over fp32, bf16 and 8-bit pools.
#include <limits.h>
#include <math.h>

#include "pool_attn_simt.cuh"

namespace wm {
namespace {

using namespace pool;

// ---------------------------------------------------------------- joining the pieces of a segment
// Block (i, j) joins rows 8 j .. of the segment that share i began and left unfinished, if its note names one.
constexpr int kJoinRows = 8, kJoinThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) pool_attn_join_kernel(const wm_pool_attn_args a, const Plan plan) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched ahead of the first kernel's end
  const int shares = gridDim.x, first = blockIdx.x;
  const Note note = *note_of(a, first);
  if (note.last < 0) return;
  const int rows = min(plan.rows_per_block, kJoinRows), per_row = kJoinThreads / rows;
  const int r = blockIdx.y * rows + threadIdx.x / per_row;
  int token, head;
  row_place(a, plan, note.kv_head, note.row_block, r, token, head);
  if (token >= a.q_len) return;
  const long long pitch = 2ll * plan.rows_per_block * (a.head_dim + 2);  // between the records of consecutive shares
  const float* begun = partial_row(a, plan, shares, first, 1, r);
  const float* rest = partial_row(a, plan, shares, first, 0, r);
  T* out = static_cast<T*>(a.out) + note.b * a.out_strides[0] + head * a.out_strides[1] + token * a.out_strides[2];
  for (int d = 2 * (threadIdx.x % per_row); d < a.head_dim; d += 2 * per_row) {
    // the running mean of the records so far; kBatch records in flight
    float top = -INFINITY, l = 0.f;
    float2 acc = make_float2(0.f, 0.f);
    constexpr int kBatch = 4;
    for (int n = 0; n <= note.last - first; n += kBatch) {
      float2 ml[kBatch], y[kBatch];
      float both = top;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const bool there = n + i <= note.last - first;
        const float* row = n + i == 0 ? begun : rest + (n + i) * pitch;
        ml[i] = there ? *reinterpret_cast<const float2*>(row) : make_float2(-INFINITY, 0.f);
        y[i] = there ? *reinterpret_cast<const float2*>(row + 2 + d) : make_float2(0.f, 0.f);
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) both = fmaxf(both, ml[i].x);
      const float ref = both == -INFINITY ? 0.f : both, keep = exp2f(top - ref);
      l *= keep;
      acc.x *= keep;
      acc.y *= keep;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float f = exp2f(ml[i].x - ref);
        l = fmaf(ml[i].y, f, l);
        acc.x = fmaf(y[i].x, f, acc.x);
        acc.y = fmaf(y[i].y, f, acc.y);
      }
      top = both;
    }
    out[d] = from_float<T>(l == 0.f ? 0.f : acc.x / l);
    out[d + 1] = from_float<T>(l == 0.f ? 0.f : acc.y / l);
  }
}

// ---------------------------------------------------------------- host
constexpr int kSms = 148;

long long rows_of(const wm_pool_attn_args& a) { return static_cast<long long>(a.q_heads / a.kv_heads) * a.q_len; }

// More than 16 rows per KV head share the pool rows of a block through shared memory.
bool in_shared(const wm_pool_attn_args& a) { return a.dtype == WM_BF16 && rows_of(a) > 16; }

int rows_per_block(const wm_pool_attn_args& a) {
  const long long rows = rows_of(a);
  return a.dtype == WM_F32 ? (rows == 1 ? 1 : rows <= 4 ? 4 : rows <= 8 ? 8 : 16) : in_shared(a) ? shared_rows_per_block(rows, a.storage, a.head_dim) : rows <= 8 ? 8 : 16;
}

// One wave: as many shares as blocks fit the GPU, and no more than there can be units.
int count_shares(const wm_pool_attn_args& a, const Plan& p) {
  const double tiles = static_cast<double>((a.k_len + kTileKeys - 1) / kTileKeys + p.draft_tiles + p.segment_cost) * a.batch * a.kv_heads * p.row_blocks;
  const int wave = kSms * (a.dtype == WM_F32 ? simt_resident_blocks(p.rows_per_block) : in_shared(a) ? 2 : resident_blocks(a.storage, p.rows_per_block / 8, a.head_dim));
  return tiles < wave ? (tiles < 1 ? 1 : static_cast<int>(tiles)) : wave;
}

// A cluster per segment where all clusters fit one wave and no block gets more than four tiles of the longest sequence the
// pool can hold: one launch instead of two, 5.7 us against 7.6 us on one sequence of 480 tokens with 16 heads.
int cluster_size(const wm_pool_attn_args& a, const Plan& p) {
  if (a.dtype == WM_F32 || p.rows_per_block > 16) return 0;
  const int tiles = (a.k_len + kTileKeys - 1) / kTileKeys + p.draft_tiles;
  int size = 1;
  while (size < kMaxCluster && size < tiles) size *= 2;
  const double blocks = static_cast<double>(a.batch) * a.kv_heads * p.row_blocks * size;
  return tiles <= 4 * size && blocks <= kSms * resident_blocks(a.storage, p.rows_per_block / 8, a.head_dim) ? size : 0;
}

bool make_plan(const wm_pool_attn_args& a, Plan& p) {
  const long long rows = rows_of(a);
  p.rows_per_block = rows_per_block(a);
  // measured with 1, 2, 4, 8.  Shared memory, heads of 64: 64 sequences with 32 drafted tokens over bf16 243, 223, 197, 201 us, over int8 328, 309,
  // 294, 304 us; small calls differ less (8 sequences with 41 tokens, 4 heads per KV head, int8: 60, 61, 65, 73 us; 24 sequences with 7, e4m3: 52, 47,
  // 49, 56 us).  Heads of 128, the same four: 223, 224, 229, 238; 274, 276, 282, 294; 106, 112, 117, 132; 76, 77, 83, 94 us.  Few rows: one token,
  // 64 sequences, int8 rows of 64 125, 125, 128, 132 us, rows of 128 with 4 heads per KV head 128, 130, 135, 145 us; fp32, 8 tokens 85, 86, 92, 99 us
  p.segment_cost = in_shared(a) ? (a.head_dim <= 64 ? 4 : 1) : 2;
  const long long blocks = (rows + p.rows_per_block - 1) / p.rows_per_block;
  p.draft_tiles = a.ancestors != nullptr ? (a.q_len + kTileKeys - 1) / kTileKeys : 0;
  p.group = a.q_heads / a.kv_heads;
  const double units = (static_cast<double>(a.k_len) / kTileKeys + 2 + p.segment_cost + p.draft_tiles) * a.batch * a.kv_heads * blocks;
  if (units >= INT_MAX || rows > INT_MAX) return false;  // the kernels count in 32 bits
  p.row_blocks = static_cast<int>(blocks);
  p.cluster = cluster_size(a, p);
  p.blocks = p.cluster > 0 ? a.batch * a.kv_heads * p.row_blocks * p.cluster : count_shares(a, p);
  return true;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned16(const int64_t* strides, int esize) {
  return strides[0] * esize % 16 == 0 && strides[1] * esize % 16 == 0 && strides[2] * esize % 16 == 0;
}

int validate(const wm_pool_attn_args& a, Plan& plan) {
  const char* who = "wm_pool_attn";
  if (a.q == nullptr || a.k == nullptr || a.v == nullptr || a.out == nullptr) return fail(WM_EINVAL, "%s: q, k, v and out are required", who);
  if (a.dtype != WM_F32 && a.dtype != WM_BF16) return fail(WM_EINVAL, "%s: dtype must be WM_F32 or WM_BF16", who);
  const bool quantised = a.storage == WM_INT8 || a.storage == WM_E4M3;
  if (!quantised && a.storage != a.dtype) return fail(WM_EINVAL, "%s: the pool must be WM_INT8, WM_E4M3 or of the queries' type", who);
  if (quantised && (a.k_scales == nullptr || a.v_scales == nullptr)) return fail(WM_EINVAL, "%s: an 8-bit pool needs its scales", who);
  if (a.batch < 1 || a.q_heads < 1 || a.kv_heads < 1 || a.q_len < 1 || a.k_len < 1 || a.head_dim < 1) return fail(WM_EINVAL, "%s: sizes must be positive", who);
  if (a.q_heads % a.kv_heads) return fail(WM_EINVAL, "%s: q_heads must be a multiple of kv_heads", who);
  if (a.lead != 0 && a.lead != 1) return fail(WM_EINVAL, "%s: lead must be 0 or 1", who);
  const int have = (a.draft_k != nullptr) + (a.draft_v != nullptr) + (a.ancestors != nullptr) + (a.depths != nullptr);
  if (have != 0 && have != 4) return fail(WM_EINVAL, "%s: drafted tokens need their keys, values and both tree tables", who);
  if (have != 0 && a.q_len > kMaxTreeNodes) return fail(WM_EUNSUPPORTED, "%s: at most %d drafted tokens", who, kMaxTreeNodes);
  const int wide = a.dtype == WM_F32 ? 4 : 2, held = quantised ? 1 : wide;
  if (a.head_dim > 128 || a.head_dim * held % 16 || a.head_dim * wide % 16) return fail(WM_EUNSUPPORTED, "%s: head_dim rows must be a multiple of 16 bytes, head_dim at most 128", who);
  if (!aligned16(a.q) || !aligned16(a.k) || !aligned16(a.v) || !aligned16(a.q_strides, wide) || !aligned16(a.k_strides, held) || !aligned16(a.v_strides, held) ||
      (have != 0 && (!aligned16(a.draft_k) || !aligned16(a.draft_v) || !aligned16(a.draft_k_strides, wide) || !aligned16(a.draft_v_strides, wide))))
    return fail(WM_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
  for (const int64_t* strides : {a.k_strides, a.v_strides, a.k_scale_strides, a.v_scale_strides})
    if (strides[2] < 0 || strides[2] >= 1 << 24) return fail(WM_EUNSUPPORTED, "%s: pool rows must be less than 2^24 elements apart", who);
  if (!aligned16(a.out) || !aligned16(a.out_strides, wide) || !aligned16(a.workspace)) return fail(WM_EUNSUPPORTED, "%s: output rows and workspace must be 16-byte aligned", who);
  if (a.k_len > kMaxSlots) return fail(WM_EUNSUPPORTED, "%s: too many slots", who);
  if (!make_plan(a, plan)) return fail(WM_EUNSUPPORTED, "%s: too many query rows", who);
  return WM_OK;
}

}  // namespace

size_t pool_attn_workspace(const wm_pool_attn_args& a) {
  Plan plan;
  if (a.batch < 1 || a.kv_heads < 1 || a.q_heads < a.kv_heads || a.q_len < 1 || a.k_len < 1 || a.k_len > kMaxSlots || !make_plan(a, plan)) return 0;
  if (plan.cluster > 0) return 0;
  return static_cast<size_t>(plan.blocks) * (sizeof(Note) + 2 * plan.rows_per_block * (a.head_dim + 2) * sizeof(float));
}

int pool_attn_launch(const wm_pool_attn_args& a, cudaStream_t stream) {
  Plan plan;
  const int status = validate(a, plan);
  if (status != WM_OK) return status;
  const size_t need = pool_attn_workspace(a);
  if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need)) return fail(WM_EWORKSPACE, "wm_pool_attn needs %zu workspace bytes, got %zu", need, a.workspace_bytes);
  const bool tree = a.ancestors != nullptr;
  cudaError_t launched;
  if (in_shared(a))
    launched = a.storage == WM_INT8 ? launch_shared<WM_INT8>(a, plan, stream) : a.storage == WM_E4M3 ? launch_shared<WM_E4M3>(a, plan, stream) : launch_shared<WM_BF16>(a, plan, stream);
  else if (a.dtype == WM_F32)
    launched = a.storage == WM_INT8 ? launch_simt<WM_INT8>(a, plan, stream) : a.storage == WM_E4M3 ? launch_simt<WM_E4M3>(a, plan, stream) : launch_simt<WM_F32>(a, plan, stream);
  else if (a.storage == WM_INT8)
    launched = tree ? launch_mma_storage<WM_INT8, true>(a, plan, stream) : launch_mma_storage<WM_INT8, false>(a, plan, stream);
  else if (a.storage == WM_E4M3)
    launched = tree ? launch_mma_storage<WM_E4M3, true>(a, plan, stream) : launch_mma_storage<WM_E4M3, false>(a, plan, stream);
  else
    launched = tree ? launch_mma_storage<WM_BF16, true>(a, plan, stream) : launch_mma_storage<WM_BF16, false>(a, plan, stream);
  count_launch();
  WM_CUDA(launched);
  if (plan.cluster > 0 || plan.blocks == 1) return WM_OK;
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(plan.blocks, (plan.rows_per_block + kJoinRows - 1) / kJoinRows);
  config.blockDim = dim3(kJoinThreads);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  const cudaError_t status_join = a.dtype == WM_F32 ? cudaLaunchKernelEx(&config, pool_attn_join_kernel<float>, a, plan)
                                                    : cudaLaunchKernelEx(&config, pool_attn_join_kernel<__nv_bfloat16>, a, plan);
  count_launch();
  return cuda_check(status_join, "pool_attn_join_kernel");
}

}  // namespace wm

extern "C" {

size_t wm_pool_attn_workspace_bytes(const wm_pool_attn_args* a) { return a ? wm::pool_attn_workspace(*a) : 0; }

int wm_pool_attn(const wm_pool_attn_args* a, void* stream) {
  if (a == nullptr) return wm::fail(WM_EINVAL, "wm_pool_attn: null arguments");
  return wm::pool_attn_launch(*a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
