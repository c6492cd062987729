// Pool attention for fp32 queries: products and sums in fp32 on the FMA pipe, over fp32 and 8-bit pools.
//
// A block of eight warps takes R rows of a KV head over a step of kStepKeys keys, whose rows arrive in shared memory by
// asynchronous copies one step ahead.  Scores: a thread per key, part of head_dim and up to eight rows; keys lie 16 bytes more than
// their size apart, which keeps them off each other's banks.  A warp per row turns the scores into weights against the row's
// running maximum.  Values: a thread per four elements and every n-th key, all R rows in its registers; those sums meet once
// per piece of a segment.
//
// Few rows are bound by HBM, many by the reads of shared memory beside the products (16 bytes of a key serve eight rows at
// most, 16 bytes of a query one key).  8 sequences of up to 8192 fp32 rows of 64, 16 heads: one token 52 us (5 130 GB/s), 8 drafted
// tokens 85 us, 16 153 us (14 TFLOP/s).  Rows per thread, on 8 sequences of up to 4100 fp32 rows of 128 with 16 tokens and 4
// heads per KV head: 4, 8, 16 take 332, 282, 424 us.
#pragma once

#include "pool_attn_shared.cuh"

namespace wm {
namespace pool {

template <int kStorage, int DP>
struct SimtCfg {
  static constexpr int kBytes = kStorage == WM_F32 ? 4 : 1;
  static constexpr int kPitch = DP * kBytes + 16;
  static constexpr int kStepKeys = kStorage == WM_F32 ? (DP == 128 ? 32 : 64) : (DP == 128 ? 64 : 128);
  static constexpr int kTileBytes = kStepKeys * kPitch;
  static constexpr int kChunks = DP * kBytes / 16;
  static constexpr int kPasses = kStepKeys * kChunks / kBlockThreads;
  static constexpr int kPassRows = kBlockThreads / kChunks;
  // drafted tokens are fp32 rows whatever the pool holds
  static constexpr int kDraftPitch = DP * 4 + 16;
  static constexpr int kDraftKeys = kStorage == WM_F32 ? kStepKeys : (DP == 128 ? 16 : 32);
  static_assert(kDraftKeys * kDraftPitch <= kTileBytes, "a step of drafted tokens fits the place of a step of the pool");
};

template <int kStorage, int DP, int R>
struct SimtShared {
  using C = SimtCfg<kStorage, DP>;
  union {
    unsigned char tile[2][2][C::kTileBytes];  // K, V of a step
    float acc[kBlockWarps][R][DP];            // at the end of a piece
  };
  float q[R][DP];
  alignas(16) float p[C::kStepKeys][R];
  float s[R][C::kStepKeys];
  float scale[kStorage == WM_F32 ? 1 : 2][2][C::kStepKeys];
  unsigned char seen[2][C::kStepKeys];
  alignas(16) float keep[R];
  float m[R], l[R];
  int token[R];  // -1: no such row, or a padding node
};
static_assert(sizeof(SimtShared<WM_F32, 64, 8>) <= 233472 / 3 - 1024 && sizeof(SimtShared<WM_F32, 128, 8>) <= 233472 / 3 - 1024, "three blocks per SM");

// Blocks of an SM: the accumulators of 16 rows leave room for two.
__host__ __device__ constexpr int simt_resident_blocks(int rows) { return rows == 16 ? 2 : 3; }

// four elements of a row in shared memory
template <int kHeld>
__device__ __forceinline__ void held_four(const unsigned char* p, float (&x)[4]) {
  if (kHeld == WM_F32) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    codes_to_float(*reinterpret_cast<const uint32_t*>(p), kHeld == WM_INT8, x);
  }
}

// Asks for a step of the pool from slot j0 on.  Rows that are not visible become zeros: what they hold must not meet their zero
// weight.
template <int kStorage, int DP, int R>
__device__ __forceinline__ void simt_ask(SimtShared<kStorage, DP, R>& sm, const wm_pool_attn_args& a, const Piece& c, int stage, int j0) {
  using C = SimtCfg<kStorage, DP>;
  const int row0 = threadIdx.x / C::kChunks, part = threadIdx.x % C::kChunks;
  const uint8_t* mask = a.key_mask != nullptr ? a.key_mask + static_cast<long long>(c.b) * a.k_len : nullptr;
  if (part * 16 < a.head_dim * C::kBytes) {
    const char* k = static_cast<const char*>(a.k) + (c.b * a.k_strides[0] + c.kv_head * a.k_strides[1]) * C::kBytes + part * 16;
    const char* v = static_cast<const char*>(a.v) + (c.b * a.v_strides[0] + c.kv_head * a.v_strides[1]) * C::kBytes + part * 16;
    const uint32_t to = ptx::smem_u32(sm.tile[stage][0]) + row0 * C::kPitch + part * 16;
#pragma unroll
    for (int n = 0; n < C::kPasses; ++n) {
      const long long j = j0 + row0 + n * C::kPassRows;
      const bool live = j < c.slots && (mask == nullptr || mask[j] != 0);
      cp_async_16(to + n * C::kPassRows * C::kPitch, live ? k + j * a.k_strides[2] * C::kBytes : static_cast<const char*>(a.k), live);
      cp_async_16(to + n * C::kPassRows * C::kPitch + C::kTileBytes, live ? v + j * a.v_strides[2] * C::kBytes : static_cast<const char*>(a.k), live);
    }
  }
  for (int i = threadIdx.x; i < C::kStepKeys; i += kBlockThreads) {
    const long long j = j0 + i;
    const bool live = j < c.slots && (mask == nullptr || mask[j] != 0);
    sm.seen[stage][i] = live;
    if (kStorage != WM_F32) {
      ptx::cp_async_4(&sm.scale[stage][0][i], live ? a.k_scales + c.b * a.k_scale_strides[0] + c.kv_head * a.k_scale_strides[1] + j * a.k_scale_strides[2] : a.k_scales, live);
      ptx::cp_async_4(&sm.scale[stage][1][i], live ? a.v_scales + c.b * a.v_scale_strides[0] + c.kv_head * a.v_scale_strides[1] + j * a.v_scale_strides[2] : a.v_scales, live);
    }
  }
}

// A step of drafted tokens from node n0 on; padding nodes may hold anything and become zeros.
template <int kStorage, int DP, int R>
__device__ __forceinline__ void simt_ask_drafts(SimtShared<kStorage, DP, R>& sm, const wm_pool_attn_args& a, const Piece& c, int stage, int n0) {
  using C = SimtCfg<kStorage, DP>;
  const int* depths = a.depths + (a.shared_tree ? 0ll : static_cast<long long>(c.b) * a.q_len);
  const int pieces = a.head_dim / 4;
  for (int i = threadIdx.x; i < C::kDraftKeys * pieces; i += kBlockThreads) {
    const int row = i / pieces, part = i - row * pieces;
    const long long j = n0 + row;
    const bool live = j < a.q_len && depths[j] >= 0;
    const float* k = static_cast<const float*>(a.draft_k) + c.b * a.draft_k_strides[0] + c.kv_head * a.draft_k_strides[1];
    const float* v = static_cast<const float*>(a.draft_v) + c.b * a.draft_v_strides[0] + c.kv_head * a.draft_v_strides[1];
    const uint32_t to = ptx::smem_u32(sm.tile[stage][0]) + row * C::kDraftPitch + part * 16;
    cp_async_16(to, live ? k + j * a.draft_k_strides[2] + part * 4 : k, live);
    cp_async_16(to + C::kTileBytes, live ? v + j * a.draft_v_strides[2] + part * 4 : v, live);
  }
}

// The scores, weights and sums of a step whose rows lie in `stage`; `there` of its keys exist.
template <int kStorage, int DP, int R, bool kDraft>
__device__ __forceinline__ void simt_step(SimtShared<kStorage, DP, R>& sm, const wm_pool_attn_args& a, const Piece& c, int stage, int j0, int there, float (&acc)[R][4]) {
  using C = SimtCfg<kStorage, DP>;
  constexpr int kHeld = kDraft ? WM_F32 : kStorage, kBytes = kHeld == WM_F32 ? 4 : 1;
  constexpr int kKeys = kDraft ? C::kDraftKeys : C::kStepKeys, kPitch = kDraft ? C::kDraftPitch : C::kPitch;
  // The threads of a key: kSets with kEach rows each, and in a set kParts with every kParts-th 16 bytes of the key's row.  They
  // lie so that eight lanes read eight different banks.
  constexpr int kPerKey = kBlockThreads / kKeys, kEach = R < 8 ? R : 8, kSets = kPerKey < R / kEach ? kPerKey : R / kEach;
  constexpr int kRows = R / kSets, kParts = kPerKey / kSets, kSide = kParts < 8 ? 32 / kParts : 1, kMine = kRows > kParts ? kRows / kParts : 1;
  constexpr int LPK = DP / 4, kSlices = kBlockThreads / LPK;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  {
    const int part = lane / kSide % kParts, key = warp % (kBlockWarps / kSets) * (32 / kParts) + (kParts < 8 ? lane % kSide : lane / kParts);
    const unsigned char* row = sm.tile[stage][0] + key * kPitch;
    int first = warp / (kBlockWarps / kSets) * kRows;
    float d[kRows] = {};
#pragma unroll kBytes == 4 ? 2 : 1
    for (int e = part * (16 / kBytes); e < a.head_dim; e += kParts * (16 / kBytes)) {
      const uint4 held = *reinterpret_cast<const uint4*>(row + e * kBytes);
      const uint32_t word[4] = {held.x, held.y, held.z, held.w};
#pragma unroll
      for (int u = 0; u < 4 / kBytes; ++u) {
        float x[4];
        if (kHeld == WM_F32) {
#pragma unroll
          for (int n = 0; n < 4; ++n) x[n] = __uint_as_float(word[n]);
        } else {
          codes_to_float(word[u], kHeld == WM_INT8, x);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float4 y = *reinterpret_cast<const float4*>(&sm.q[first + r][e + 4 * u]);
          d[r] = fmaf(x[0], y.x, d[r]);
          d[r] = fmaf(x[1], y.y, d[r]);
          d[r] = fmaf(x[2], y.z, d[r]);
          d[r] = fmaf(x[3], y.w, d[r]);
        }
      }
    }
    // the parts' sums, each lane keeping its share of the rows: rows `first` .. first + kMine - 1
    __syncwarp();
#pragma unroll
    for (int o = 1, n = kRows; o < kParts; o *= 2) {
      const int to = o * kSide;
      if (n > 1) {
        n /= 2;
        const bool high = lane & to;
#pragma unroll
        for (int i = 0; i < n; ++i) {
          const float other = high ? d[i] : d[n + i];
          d[i] = (high ? d[n + i] : d[i]) + __shfl_xor_sync(0xffffffffu, other, to);
        }
        first += high ? n : 0;
      } else {
        d[0] += __shfl_xor_sync(0xffffffffu, d[0], to);
      }
    }
    float factor = a.scale * kLog2e;
    if (kHeld != WM_F32) factor *= sm.scale[kHeld != WM_F32 ? stage : 0][0][key];
    const bool seen = kDraft ? key < there : sm.seen[stage][key] != 0;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int r = first + i;
      bool use = seen;
      if (kDraft && seen) {
        const int token = sm.token[r], words = (a.q_len + 31) / 32, j = j0 + key;
        use = token >= 0 && (a.ancestors[((a.shared_tree ? 0ll : static_cast<long long>(c.b) * a.q_len) + token) * words + (j >> 5)] >> (j & 31) & 1u);
      }
      sm.s[r][key] = use ? d[i] * factor : -INFINITY;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int r = warp; r < R; r += kBlockWarps) {
    constexpr int kKeysEach = kKeys > 32 ? kKeys / 32 : 1;
    const float before = sm.m[r];
    float x[kKeysEach], top = before;
#pragma unroll
    for (int i = 0; i < kKeysEach; ++i) {
      x[i] = lane < kKeys ? sm.s[r][lane + 32 * i] : -INFINITY;
      top = fmaxf(top, x[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(before - ref);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kKeysEach; ++i) {
      const int key = lane + 32 * i;
      const float p = exp2f(x[i] - ref);
      sum += p;
      // -1: a drafted token that the row does not see, whose value may be anything
      if (lane < kKeys) sm.p[key][r] = kDraft ? (x[i] == -INFINITY ? -1.f : p) : kHeld == WM_F32 ? p : p * sm.scale[kHeld != WM_F32 ? stage : 0][1][key];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      sm.keep[r] = keep;
      sm.m[r] = top;
      sm.l[r] = fmaf(sm.l[r], keep, sum);
    }
  }
  __syncthreads();
  const auto rows4 = [](const float* from, int r) {
    if (R == 1) return make_float4(from[0], 0.f, 0.f, 0.f);
    return *reinterpret_cast<const float4*>(from + r);
  };
#pragma unroll
  for (int r = 0; r < R; r += 4) {
    const float4 keep = rows4(sm.keep, r);
    const float f[4] = {keep.x, keep.y, keep.z, keep.w};
#pragma unroll
    for (int i = 0; i < 4 && r + i < R; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r + i][e] *= f[i];
  }
  const int d0 = lane % LPK * 4;
  if (d0 < a.head_dim) {
    const unsigned char* rows = sm.tile[stage][1] + d0 * kBytes;
#pragma unroll 4
    for (int key = warp * (32 / LPK) + lane / LPK; key < min(kKeys, there); key += kSlices) {
      float y[4];
      held_four<kHeld>(rows + key * kPitch, y);
#pragma unroll
      for (int r = 0; r < R; r += 4) {
        const float4 w = rows4(sm.p[key], r);
        const float p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4 && r + i < R; ++i) {
          if (kDraft && p[i] < 0.f) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r + i][e] = fmaf(p[i], y[e], acc[r + i][e]);
        }
      }
    }
  }
}

template <int kStorage, int DP, int R>
__global__ void __launch_bounds__(kBlockThreads, simt_resident_blocks(R)) pool_attn_simt_kernel(const wm_pool_attn_args a, const Plan plan) {
  using C = SimtCfg<kStorage, DP>;
  constexpr int LPK = DP / 4;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  SimtShared<kStorage, DP, R>& sm = *reinterpret_cast<SimtShared<kStorage, DP, R>*>(smem_raw);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may take its place: it waits for this one's end
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Share share = find_share(a, plan, blockIdx.x, gridDim.x);
  if (tid == 0) note_of(a, blockIdx.x)->last = -1;
  for (int at = share.begin; at < share.end;) {
    const Piece c = next_piece(a, plan, at, share.end, share.b, share.b_begin);
    at = c.end;
    if (c.tile >= c.stop) continue;
    const int past_end = min(c.slots, c.stop * kTileKeys), first_key = c.tile * kTileKeys;
    const int past_steps = c.tile < c.past_tiles ? (past_end - first_key + C::kStepKeys - 1) / C::kStepKeys : 0;
    const int first_node = max(c.tile - c.past_tiles, 0) * kTileKeys;
    const int draft_steps =
        a.ancestors != nullptr && c.stop > c.past_tiles ? (min(a.q_len, (c.stop - c.past_tiles) * kTileKeys) - first_node + C::kDraftKeys - 1) / C::kDraftKeys : 0;
    const int steps = past_steps + draft_steps;
    const auto ask = [&](int i) {
      if (i < past_steps)
        simt_ask(sm, a, c, i & 1, first_key + i * C::kStepKeys);
      else if (i < steps)
        simt_ask_drafts(sm, a, c, i & 1, first_node + (i - past_steps) * C::kDraftKeys);
      ptx::cp_async_commit();
    };
    ask(0);
    for (int i = tid; i < R * LPK; i += kBlockThreads) {
      const int r = i / LPK, d = i % LPK * 4;
      int token, head;
      row_place(a, plan, c.kv_head, c.row_block, r, token, head);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (token < a.q_len && d < a.head_dim)
        x = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + c.b * a.q_strides[0] + head * a.q_strides[1] + token * a.q_strides[2] + d);
      *reinterpret_cast<float4*>(&sm.q[r][d]) = x;
    }
    if (tid < R) {
      int token, head;
      row_place(a, plan, c.kv_head, c.row_block, tid, token, head);
      if (token >= a.q_len) token = -1;
      if (token >= 0 && a.depths != nullptr && a.depths[(a.shared_tree ? 0ll : static_cast<long long>(c.b) * a.q_len) + token] < 0) token = -1;
      sm.token[tid] = token;
      sm.m[tid] = -INFINITY;
      sm.l[tid] = 0.f;
    }
    float acc[R][4] = {};
#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      cp_async_wait<0>();
      __syncthreads();  // step i is there for every warp, and step i - 1 has been read by every warp
      ask(i + 1);
      if (i < past_steps)
        simt_step<kStorage, DP, R, false>(sm, a, c, i & 1, first_key + i * C::kStepKeys, c.slots - first_key - i * C::kStepKeys, acc);
      else
        simt_step<kStorage, DP, R, true>(sm, a, c, i & 1, first_node + (i - past_steps) * C::kDraftKeys, a.q_len - first_node - (i - past_steps) * C::kDraftKeys, acc);
    }
    cp_async_wait<0>();
    __syncthreads();
    // the sums of a warp's lanes, then of the warps
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int o = LPK; o < 32; o <<= 1) acc[r][e] += __shfl_xor_sync(0xffffffffu, acc[r][e], o);
      }
      if (lane < LPK) *reinterpret_cast<float4*>(&sm.acc[warp][r][lane * 4]) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
    }
    __syncthreads();
    for (int i = tid; i < R * a.head_dim; i += kBlockThreads) {
      const int r = i / a.head_dim, d = i - r * a.head_dim;
      int token, head;
      row_place(a, plan, c.kv_head, c.row_block, r, token, head);
      if (token >= a.q_len) continue;
      const bool empty = sm.token[r] < 0 || sm.l[r] == 0.f;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kBlockWarps; ++w) sum += sm.acc[w][r][d];
      if (whole(c)) {
        static_cast<float*>(a.out)[c.b * a.out_strides[0] + head * a.out_strides[1] + token * a.out_strides[2] + d] = empty ? 0.f : sum / sm.l[r];
      } else {
        float* row = partial_row(a, plan, gridDim.x, blockIdx.x, c.tile == 0, r);
        if (d == 0) row[0] = empty ? -INFINITY : sm.m[r], row[1] = empty ? 0.f : sm.l[r];
        row[2 + d] = empty ? 0.f : sum;
      }
    }
    if (tid == 0) leave_note(a, share, c, blockIdx.x, gridDim.x);
    __syncthreads();
  }
}

template <int kStorage, int DP, int R>
cudaError_t launch_simt_rows(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {
  constexpr int kBytes = static_cast<int>(sizeof(SimtShared<kStorage, DP, R>));
  static DeviceFlags done;
  const cudaError_t error = opt_in(pool_attn_simt_kernel<kStorage, DP, R>, kBytes, done);
  if (error != cudaSuccess) return error;
  pool_attn_simt_kernel<kStorage, DP, R><<<plan.blocks, kBlockThreads, kBytes, stream>>>(a, plan);
  return cudaGetLastError();
}

template <int kStorage, int DP>
cudaError_t launch_simt_dim(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {
  switch (plan.rows_per_block) {
    case 1: return launch_simt_rows<kStorage, DP, 1>(a, plan, stream);
    case 4: return launch_simt_rows<kStorage, DP, 4>(a, plan, stream);
    case 8: return launch_simt_rows<kStorage, DP, 8>(a, plan, stream);
    default: return launch_simt_rows<kStorage, DP, 16>(a, plan, stream);
  }
}

// One translation unit per way of holding the pool.
template <int kStorage>
cudaError_t launch_simt(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream);

#define WM_POOL_SIMT_UNIT(kStorage)                                                                       \
  template <>                                                                                             \
  cudaError_t launch_simt<kStorage>(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {  \
    if (a.head_dim <= 32) return launch_simt_dim<kStorage, 32>(a, plan, stream);                          \
    if (a.head_dim <= 64) return launch_simt_dim<kStorage, 64>(a, plan, stream);                          \
    return launch_simt_dim<kStorage, 128>(a, plan, stream);                                               \
  }

}  // namespace pool
}  // namespace wm
