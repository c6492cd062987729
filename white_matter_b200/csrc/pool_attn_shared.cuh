// Pool attention for bf16 queries with more than 16 rows per KV head (trees of drafted tokens, grouped heads, chunks of new
// tokens): the same transposed products on the warp-level matrix instructions as pool_attn_mma.cuh, with the pool rows in
// shared memory, where all rows of the block use them.
//
// A block of eight warps holds 16 rows per warp: kRowGroups warps side by side cover the rows, 8 / kRowGroups such sets share
// the keys of a step.  16 rows keep a warp's accumulators small, so two blocks fit an SM; the registers of one warp for 32
// rows (its rows' accumulators beside the pool rows in flight) left 12 warps per SM, which hid too little latency
// (IPC 1.35 on 64 sequences with 32 drafted tokens, 250 us; this kernel: 198 us, 5 490 GB/s).
//
// A step is 128 keys (heads of up to 64) or 64 keys, as bf16 rows of DP elements.  bf16 rows arrive by asynchronous copies, two steps ahead; 8-bit
// rows by the same copies, one step ahead, into a corner of the thread that turns their codes into bf16.  Rows that are not visible are
// stored as zeros.
//
// Weights, times the value's scale, are rounded to bf16 and summed as rounded: results are up to 1.4 times as far from the exact ones
// as the output's own rounding (1.1 to 1.2 over bf16 and e4m3 pools).  The second part that the register kernel takes would double
// the products of the values.
//
// Heads of less than 64 are computed as 64 and of 72 to 120 as 128: 24 sequences of up to 5000 int8 rows, 32 rows per KV head, take 45, 46, 48, 46 us with
// heads of 16, 32, 48, 64 and 73, 73, 76, 72 us with 80, 96, 112, 128.  The kernels with drafted tokens over 8-bit rows of 128 spill (128
// registers; 120 bytes of spill stores for int8, 24 without drafted tokens).
#pragma once

#include <atomic>

#include "pool_attn_mma.cuh"

namespace wm {
namespace pool {

constexpr int kBlockWarps = 8, kBlockThreads = kBlockWarps * 32;

// Rows in shared memory, so that the eight rows of a matrix keep off each other's banks: wide ones 16 bytes apart, narrow ones
// without a gap, their 16-byte pieces permuted by the row (piece ^ row % 8).  A gap costs no instruction where the permutation
// costs one per matrix (8 sequences with 41 drafted tokens, 4 heads of 128 per KV head, int8: 106 us against 110 us); a gap in rows of
// 64 cost more than it gave (64 sequences with 32 drafted tokens, bf16: some 5 % slower).
template <int DP>
struct RowLayout {
  static constexpr bool kPermuted = DP == 64;
  static constexpr int kPitch = DP * 2 + (kPermuted ? 0 : 16);
  __device__ static uint32_t piece(int row, int piece) { return row * kPitch + ((kPermuted ? piece ^ (row & 7) : piece) << 4); }
  // the piece 2 s behind the one that `at` names, which is piece 0 or 1 of a row in a buffer aligned to its rows
  __device__ static uint32_t behind(uint32_t at, int s) { return kPermuted ? at ^ (s << 5) : at + (s << 5); }
};

template <int kStorage, int DP>
struct SharedCfg {
  static constexpr int kBytes = kStorage == WM_BF16 ? 2 : 1;
  static constexpr int kStepKeys = DP == 64 ? 128 : 64;
  static constexpr int kStages = kStorage == WM_BF16 && DP == 64 ? 3 : 2;
  static constexpr int kRowBytes = RowLayout<DP>::kPitch;
  static constexpr int kTileBytes = kStepKeys * kRowBytes;
  static constexpr int kChunks = DP * kBytes / 16;                               // 16-byte pieces of a pool row
  static constexpr int kPasses = kStepKeys * kChunks / kBlockThreads;            // pieces of K (or V) per thread and step
  static constexpr int kPassRows = kBlockThreads / kChunks;
};

template <int kStorage, int DP, int kRowGroups>
struct BlockShared {
  using C = SharedCfg<kStorage, DP>;
  static constexpr int kSide = kBlockWarps / kRowGroups > 2 ? 2 : kBlockWarps / kRowGroups;
  static constexpr int kPitch = DP + 4;
  union {
    unsigned char tile[C::kStages][2][C::kTileBytes];    // K, V of a step
    float acc[kSide][kRowGroups * 16][kPitch];           // at the end of a piece: sums of two sets of warps
  };
  uint4 raw[kStorage == WM_BF16 ? 1 : 2 * C::kPasses][kStorage == WM_BF16 ? 1 : kBlockThreads];  // a step's codes, a corner per thread
  unsigned char q[DP > 64 ? kRowGroups * 16 * C::kRowBytes : 16];
  float scale[kStorage == WM_BF16 ? 1 : C::kStages][2][C::kStepKeys];
  unsigned char seen[C::kStages][C::kStepKeys];      // key_mask of a step's rows
  float m[kBlockWarps / kRowGroups][kRowGroups * 16], l[kBlockWarps / kRowGroups][kRowGroups * 16];
  int poison[2];  // the drafted values of this piece, and of the next, hold an infinity or NaN
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void st_shared_16(uint32_t dst, const uint4& x) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_16(uint32_t src) {
  uint4 x;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(src) : "memory");
  return x;
}
__device__ __forceinline__ uint4 load_16(const char* p) {
  uint4 x;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p));
  return x;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t src) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(src) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t src) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(src) : "memory");
}
// Elements 4i .. 4i + 3 in the order 0, 2, 1, 3: how a word of codes comes apart, and so how 8-bit kernels hold every row
__device__ __forceinline__ uint4 permuted(const uint4& x) {
  return make_uint4(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632), __byte_perm(x.z, x.w, 0x5410), __byte_perm(x.z, x.w, 0x7632));
}
__device__ __forceinline__ uint32_t finite_halves(uint32_t x, bool& special) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u, special = true;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu, special = true;
  return x;
}

// ---------------------------------------------------------------- pool rows to shared memory
template <int kStorage, int DP, int kRowGroups>
struct Stager {
  using C = SharedCfg<kStorage, DP>;
  BlockShared<kStorage, DP, kRowGroups>& sm;
  const wm_pool_attn_args& a;
  const Piece& c;
  const char *k, *v;  // this thread's part of the piece's first step
  const uint8_t* mask;
  uint32_t k_pass, v_pass;
  bool inside;
  const int turn;  // parity of the piece

  __device__ Stager(BlockShared<kStorage, DP, kRowGroups>& shared, const wm_pool_attn_args& args, const Piece& piece, int parity) : sm(shared), a(args), c(piece), turn(parity) {
    const int row = threadIdx.x / C::kChunks, part = threadIdx.x % C::kChunks;
    const long long j = static_cast<long long>(c.tile) * kTileKeys + row;
    k = static_cast<const char*>(a.k) + (c.b * a.k_strides[0] + c.kv_head * a.k_strides[1] + j * a.k_strides[2]) * C::kBytes + part * 16;
    v = static_cast<const char*>(a.v) + (c.b * a.v_strides[0] + c.kv_head * a.v_strides[1] + j * a.v_strides[2]) * C::kBytes + part * 16;
    k_pass = static_cast<uint32_t>(C::kPassRows * a.k_strides[2]) * C::kBytes;
    v_pass = static_cast<uint32_t>(C::kPassRows * a.v_strides[2]) * C::kBytes;
    inside = part * 16 < a.head_dim * C::kBytes;
    mask = a.key_mask != nullptr ? a.key_mask + static_cast<long long>(c.b) * a.k_len : nullptr;
  }
  __device__ bool live(int j) const { return inside && j < c.slots && (mask == nullptr || mask[j] != 0); }

  // Asks for step i of the piece (slots from j0 on), and moves on: bf16 rows into their stage, 8-bit rows into the thread's
  // corner; called when the stage's last reader is through.
  __device__ void ask(int i, int j0) {
    const int row0 = threadIdx.x / C::kChunks, part = threadIdx.x % C::kChunks;
    if (inside) {
      const uint32_t to = kStorage == WM_BF16 ? ptx::smem_u32(sm.tile[i % C::kStages][0]) + RowLayout<DP>::piece(row0, part)
                                              : ptx::smem_u32(&sm.raw[0][kStorage == WM_BF16 ? 0 : threadIdx.x]);
      constexpr int kStep = kStorage == WM_BF16 ? C::kPassRows * C::kRowBytes : kBlockThreads * 16, kValues = kStorage == WM_BF16 ? C::kTileBytes : C::kPasses * kStep;
      if (mask == nullptr && j0 + C::kStepKeys <= c.slots) {
#pragma unroll
        for (int p = 0; p < C::kPasses; ++p) cp_async_16(to + p * kStep, k + p * k_pass);
#pragma unroll
        for (int p = 0; p < C::kPasses; ++p) cp_async_16(to + p * kStep + kValues, v + p * v_pass);
      } else {
        bool yes[C::kPasses];
#pragma unroll
        for (int p = 0; p < C::kPasses; ++p) yes[p] = live(j0 + row0 + p * C::kPassRows);
#pragma unroll
        for (int p = 0; p < C::kPasses; ++p) {
          cp_async_16(to + p * kStep, yes[p] ? k + p * k_pass : static_cast<const char*>(a.k), yes[p]);
          cp_async_16(to + p * kStep + kValues, yes[p] ? v + p * v_pass : static_cast<const char*>(a.k), yes[p]);
        }
      }
    }
    if (kStorage != WM_BF16 && static_cast<int>(threadIdx.x) < 2 * C::kStepKeys) {
      const int value = threadIdx.x / C::kStepKeys, j = j0 + threadIdx.x % C::kStepKeys;
      const float* from = value ? a.v_scales + c.b * a.v_scale_strides[0] + c.kv_head * a.v_scale_strides[1] + j * a.v_scale_strides[2]
                                : a.k_scales + c.b * a.k_scale_strides[0] + c.kv_head * a.k_scale_strides[1] + j * a.k_scale_strides[2];
      ptx::cp_async_4(&sm.scale[i % C::kStages][value][threadIdx.x % C::kStepKeys], j < c.slots ? from : a.k_scales, j < c.slots);
    }
    if (mask != nullptr && static_cast<int>(threadIdx.x) < C::kStepKeys) {
      const int j = j0 + threadIdx.x;
      sm.seen[i % C::kStages][threadIdx.x] = j < c.slots ? mask[j] : 0;
    }
    k += C::kStepKeys * a.k_strides[2] * C::kBytes;
    v += C::kStepKeys * a.v_strides[2] * C::kBytes;
  }

  // 8-bit rows: the codes in this thread's corner as bf16 into their stage.
  __device__ void store(int i) {
    if (!inside) return;
    const int row0 = threadIdx.x / C::kChunks, part = threadIdx.x % C::kChunks;
    const uint32_t to = ptx::smem_u32(sm.tile[i % C::kStages][0]);
    const uint32_t first = to + RowLayout<DP>::piece(row0, 2 * part), second = to + RowLayout<DP>::piece(row0, 2 * part + 1);
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < 2 * C::kPasses; ++n) {
      const uint4 x = sm.raw[kStorage == WM_BF16 ? 0 : n][kStorage == WM_BF16 ? 0 : threadIdx.x];
      const int at = n % C::kPasses * C::kPassRows * C::kRowBytes + n / C::kPasses * C::kTileBytes;
      uint32_t y[8];
      Codes<kStorage>::pairs(x.x, y[0], y[1], top);
      Codes<kStorage>::pairs(x.y, y[2], y[3], top);
      Codes<kStorage>::pairs(x.z, y[4], y[5], top);
      Codes<kStorage>::pairs(x.w, y[6], y[7], top);
      st_shared_16(first + at, make_uint4(y[0], y[1], y[2], y[3]));
      st_shared_16(second + at, make_uint4(y[4], y[5], y[6], y[7]));
    }
    if (Codes<kStorage>::some_nan(top)) {  // all rows of a block see the same slots, so a NaN may go through the products
#pragma unroll 1
      for (int n = 0; n < 2 * C::kPasses; ++n) {
        const int at = n % C::kPasses * C::kPassRows * C::kRowBytes + n / C::kPasses * C::kTileBytes;
        repair(first + at);
        repair(second + at);
      }
    }
  }
  __device__ static void repair(uint32_t at) {
    uint4 y = ld_shared_16(at);
    y = make_uint4(Codes<kStorage>::repaired(y.x), Codes<kStorage>::repaired(y.y), Codes<kStorage>::repaired(y.z), Codes<kStorage>::repaired(y.w));
    st_shared_16(at, y);
  }

  // A step of drafted tokens from node n0 on, by plain loads, eight in flight per thread.  Values that are not finite become
  // zeros with a note: an infinity or NaN must reach the rows that see it, and a product would carry it to all.  (Padding
  // nodes need no care: nobody sees them, so their scores and this note are not looked at.)
  __device__ void draft(int i, int n0) {
    constexpr int kPieces = DP / 8, kTotal = 2 * C::kStepKeys * kPieces, kBatch = 8;
    bool special = false;
#pragma unroll 1
    for (int at0 = threadIdx.x; at0 < kTotal; at0 += kBatch * kBlockThreads) {
      uint4 x[kBatch];
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int at = at0 + n * kBlockThreads;
        const int value = at / (C::kStepKeys * kPieces), row = at / kPieces % C::kStepKeys, part = at % kPieces, j = n0 + row;
        x[n] = make_uint4(0, 0, 0, 0);
        if (j < a.q_len && part * 8 < a.head_dim) {
          const char* from = value ? static_cast<const char*>(a.draft_v) + (c.b * a.draft_v_strides[0] + c.kv_head * a.draft_v_strides[1] + j * a.draft_v_strides[2] + part * 8) * 2
                                   : static_cast<const char*>(a.draft_k) + (c.b * a.draft_k_strides[0] + c.kv_head * a.draft_k_strides[1] + j * a.draft_k_strides[2] + part * 8) * 2;
          x[n] = load_16(from);
        }
      }
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int at = at0 + n * kBlockThreads;
        const int value = at / (C::kStepKeys * kPieces), row = at / kPieces % C::kStepKeys, part = at % kPieces;
        uint4 y = x[n];
        if (value) y = make_uint4(finite_halves(y.x, special), finite_halves(y.y, special), finite_halves(y.z, special), finite_halves(y.w, special));
        if (kStorage != WM_BF16) y = permuted(y);
        st_shared_16(ptx::smem_u32(sm.tile[i % C::kStages][0]) + value * C::kTileBytes + RowLayout<DP>::piece(row, part), y);
      }
    }
    if (special) sm.poison[turn] = 1;
  }
};

// ---------------------------------------------------------------- a warp's 16 rows
template <int DP>
struct RowQueries {
  static constexpr bool kInRegisters = DP == 64;
  uint2 reg[kInRegisters ? 2 : 1][kInRegisters ? DP / 16 : 1];  // [tile of 8 rows][16 of head_dim]
  uint32_t shared;                                             // ldmatrix address: rows of a tile, pieces 0 .. 3
};

// U groups of 16 keys against the warp's 16 rows; `k` is the lane's address in the first of them.
template <int DP, int U>
__device__ __forceinline__ void shared_scores(const RowQueries<DP>& q, uint32_t k, float (&x)[U][2][4]) {
  constexpr int kPitch = RowLayout<DP>::kPitch;
#pragma unroll
  for (int s = 0; s < DP / 16; s += 2) {
    uint32_t b[2][4];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      if (RowQueries<DP>::kInRegisters) {
        const uint2 lo = q.reg[rt][RowQueries<DP>::kInRegisters ? s : 0], hi = q.reg[rt][RowQueries<DP>::kInRegisters ? s + 1 : 0];
        b[rt][0] = lo.x, b[rt][1] = lo.y, b[rt][2] = hi.x, b[rt][3] = hi.y;
      } else {
        // lanes 0-7, 8-15, 16-23, 24-31 name the rows of pieces 2s .. 2s + 3
        ldmatrix_x4(b[rt], RowLayout<DP>::behind(q.shared + rt * 8 * kPitch, s));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t ka[4], kb[4];
      ldmatrix_x4(ka, RowLayout<DP>::behind(k + u * 16 * kPitch, s));
      ldmatrix_x4(kb, RowLayout<DP>::behind(k + u * 16 * kPitch, s + 1));
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        if (s == 0)
          mma_16816_first(x[u][rt], ka[0], ka[1], ka[2], ka[3], b[rt][0], b[rt][1]);
        else
          mma_16816(x[u][rt], ka[0], ka[1], ka[2], ka[3], b[rt][0], b[rt][1]);
        mma_16816(x[u][rt], kb[0], kb[1], kb[2], kb[3], b[rt][2], b[rt][3]);
      }
    }
  }
}

template <int DP, int U>
__device__ __forceinline__ void shared_values(State<DP, 2>& st, uint32_t v, const uint32_t (&pb)[U][2][2]) {
  constexpr int kPitch = RowLayout<DP>::kPitch;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      uint32_t va[4];
      ldmatrix_x4_trans(va, RowLayout<DP>::behind(v + u * 16 * kPitch, s));
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) mma_16816(st.o[s][rt], va[0], va[1], va[2], va[3], pb[u][rt][0], pb[u][rt][1]);
    }
}

template <int kStorage, int DP, int kRowGroups, bool kTree>
__global__ void __launch_bounds__(kBlockThreads, 2) pool_attn_shared_kernel(const wm_pool_attn_args a, const Plan plan) {
  using C = SharedCfg<kStorage, DP>;
  constexpr bool kScaled = kStorage != WM_BF16;
  constexpr int kRows = kRowGroups * 16, kSets = kBlockWarps / kRowGroups, kSetKeys = C::kStepKeys / kSets;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  BlockShared<kStorage, DP, kRowGroups>& sm = *reinterpret_cast<BlockShared<kStorage, DP, kRowGroups>*>(smem_raw);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may take its place: it waits for this one's end
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, row_group = warp % kRowGroups, set = warp / kRowGroups;
  const float factor = a.scale * kLog2e;
  constexpr int U = DP == 64 ? 2 : 1;  // groups of 16 keys taken together: what the registers hold
  constexpr uint32_t kFull = U == 2 ? 0xffffffffu : 0xffffu;
  // ldmatrix of K: lanes 0-15 name the 16 keys' low halves of 16 elements, 16-31 the high ones; of V, transposed: lanes 0-7 and 8-15 keys
  // 0-7 (low, high), 16-23 and 24-31 keys 8-15
  const uint32_t k_lane = RowLayout<DP>::piece(lane & 15, lane >> 4), v_lane = RowLayout<DP>::piece((lane & 7) + ((lane & 16) >> 1), lane >> 3 & 1);
  if (tid == 0) {
    note_of(a, blockIdx.x)->last = -1;
    sm.poison[0] = sm.poison[1] = 0;
  }
  // columns behind head_dim are never written: zeros
  if (a.head_dim < DP) {
    for (int i = tid; i < static_cast<int>(sizeof(sm.tile) / 16); i += kBlockThreads) reinterpret_cast<uint4*>(sm.tile)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  Share share = find_share(a, plan, blockIdx.x, gridDim.x);
  int turn = 0;
  for (int at = share.begin; at < share.end;) {
    const Piece c = next_piece(a, plan, at, share.end, share.b, share.b_begin);
    at = c.end;
    if (c.tile >= c.stop) continue;

    const int past_end = min(c.slots, c.stop * kTileKeys), first_key = c.tile * kTileKeys;
    const int past_steps = c.tile < c.past_tiles ? (past_end - first_key + C::kStepKeys - 1) / C::kStepKeys : 0;
    const int first_node = max(c.tile - c.past_tiles, 0) * kTileKeys;
    const int draft_steps = kTree && c.stop > c.past_tiles ? (min(a.q_len, (c.stop - c.past_tiles) * kTileKeys) - first_node + C::kStepKeys - 1) / C::kStepKeys : 0;
    const int steps = past_steps + draft_steps;
    Stager<kStorage, DP, kRowGroups> stager(sm, a, c, turn);
    constexpr int kAhead = C::kStages - 1;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i < past_steps) stager.ask(i, first_key + i * C::kStepKeys);
      ptx::cp_async_commit();
    }

    // this warp's queries
    RowQueries<DP> q;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
      int token, head;
      if (RowQueries<DP>::kInRegisters) {
        row_place(a, plan, c.kv_head, c.row_block, row_group * 16 + rt * 8 + g, token, head);
        const char* row = static_cast<const char*>(a.q) + (token < a.q_len ? (c.b * a.q_strides[0] + head * a.q_strides[1] + token * a.q_strides[2]) * 2 : 0);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
          // elements 2t, 2t + 1 and 2t + 8, 2t + 9 of the 16; held in the order 0, 2, 1, 3 of every four for 8-bit pools
          uint2 x = make_uint2(0, 0);
          const int d = 16 * s + 2 * t;
          if (token < a.q_len) {
            if (!kScaled) {
              if (d < a.head_dim) x.x = *reinterpret_cast<const uint32_t*>(row + 2 * d);
              if (d + 8 < a.head_dim) x.y = *reinterpret_cast<const uint32_t*>(row + 2 * d + 16);
            } else {
              const int four = 16 * s + 4 * (t >> 1);
              const uint32_t pick = t & 1 ? 0x7632 : 0x5410;
              if (four < a.head_dim) {
                const uint2 y = *reinterpret_cast<const uint2*>(row + 2 * four);
                x.x = __byte_perm(y.x, y.y, pick);
              }
              if (four + 8 < a.head_dim) {
                const uint2 y = *reinterpret_cast<const uint2*>(row + 2 * four + 16);
                x.y = __byte_perm(y.x, y.y, pick);
              }
            }
          }
          q.reg[RowQueries<DP>::kInRegisters ? rt : 0][RowQueries<DP>::kInRegisters ? s : 0] = x;
        }
      }
    }
    if (!RowQueries<DP>::kInRegisters) {
      constexpr int kPieces = DP / 8;
      q.shared = ptx::smem_u32(sm.q) + row_group * 16 * C::kRowBytes + RowLayout<DP>::piece(lane & 7, lane >> 3);
      for (int i = tid; i < kRows * kPieces; i += kBlockThreads) {
        const int row = i / kPieces, part = i % kPieces;
        int token, head;
        row_place(a, plan, c.kv_head, c.row_block, row, token, head);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (token < a.q_len && part * 8 < a.head_dim)
          x = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.q) + (c.b * a.q_strides[0] + head * a.q_strides[1] + token * a.q_strides[2] + part * 8) * 2);
        if (kScaled) x = permuted(x);
        st_shared_16(ptx::smem_u32(sm.q) + RowLayout<DP>::piece(row, part), x);
      }
    }
    State<DP, 2> st;
    st.fresh = 15u;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) st.m[rt][j] = 0.f, st.l[rt][j] = 0.f;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[s][rt][e] = 0.f;
    }

#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      const bool draft = kTree && i >= past_steps;
      const int j0 = draft ? first_node + (i - past_steps) * C::kStepKeys : first_key + i * C::kStepKeys;
      cp_async_wait<kAhead - 1>();
      if (draft)
        stager.draft(i, j0);
      else if (kScaled)
        stager.store(i);
      __syncthreads();  // step i is there for every warp, and step i - 1 has been read by every warp
      if (i + kAhead < past_steps) stager.ask(i + kAhead, j0 + kAhead * C::kStepKeys);
      ptx::cp_async_commit();
      const int stage = i % C::kStages;
      const uint32_t k_rows = ptx::smem_u32(sm.tile[stage][0]) + k_lane, v_rows = ptx::smem_u32(sm.tile[stage][1]) + v_lane;
      const int there = min(kSetKeys, (draft ? a.q_len : c.slots) - j0 - set * kSetKeys);
      if (!draft) {
#pragma unroll 1
        for (int key = 0; key < there; key += 16 * U) {
          const int first = set * kSetKeys + key, left = there - key;
          uint32_t word = left >= 16 * U ? kFull : (1u << left) - 1u;
          if (a.key_mask != nullptr) word = __ballot_sync(0xffffffffu, lane < 16 * U && sm.seen[stage][first + (lane & (16 * U - 1))] != 0);
          Keys keys[U];
          uint32_t seen[U][1][2];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            keys[u].all = word == kFull;
            seen[u][0][0] = seen[u][0][1] = keys[u].all ? 3u : (word >> (16 * u + g) & 1u) | (word >> (16 * u + g + 8) & 1u) << 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              keys[u].factor[h] = kScaled ? factor * sm.scale[stage][0][first + 16 * u + g + 8 * h] : factor;
              keys[u].scale[h] = kScaled ? usable_scale(sm.scale[stage][1][first + 16 * u + g + 8 * h], keys[u].all || (seen[u][0][0] >> h & 1u)) : 1.f;
            }
          }
          float x[U][2][4];
          uint32_t pb[U][2][2];
          shared_scores<DP, U>(q, k_rows + first * C::kRowBytes, x);
          weights<DP, 2, U, kScaled, false>(st, x, keys, seen, pb);
          shared_values<DP, U>(st, v_rows + first * C::kRowBytes, pb);
        }
      } else if (kTree) {
#pragma unroll 1
        for (int key = 0; key < there; key += 16) {
          const int first = set * kSetKeys + key, words = (a.q_len + 31) / 32;
          const long long tree = a.shared_tree ? 0 : static_cast<long long>(c.b) * a.q_len;
          const Keys keys[1] = {{{factor, factor}, {1.f, 1.f}, false}};
          uint32_t seen[1][2][2];
#pragma unroll
          for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              int token, head;
              row_place(a, plan, c.kv_head, c.row_block, row_group * 16 + rt * 8 + 2 * t + j, token, head);
              const uint32_t sees = token < a.q_len ? a.ancestors[(tree + token) * words + ((j0 + first) >> 5)] >> ((j0 + first) & 31) : 0u;
              seen[0][rt][j] = (sees >> g & 1u) | (sees >> (g + 8) & 1u) << 1;
            }
          float x[1][2][4];
          uint32_t pb[1][2][2];
          shared_scores<DP, 1>(q, k_rows + first * C::kRowBytes, x);
          weights<DP, 2, 1, kScaled, true>(st, x, keys, seen, pb);
          shared_values<DP, 1>(st, v_rows + first * C::kRowBytes, pb);
        }
      }
    }

    // join the sets of warps: references and sums, then the accumulators, two sets side by side
#pragma unroll
    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = st.l[rt][j];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (st.fresh >> (2 * rt + j) & 1u) st.m[rt][j] = kNoReference;
        if (g == 0) {
          sm.m[set][row_group * 16 + rt * 8 + 2 * t + j] = st.m[rt][j];
          sm.l[set][row_group * 16 + rt * 8 + 2 * t + j] = l;
        }
      }
    __syncthreads();
    constexpr int kSide = BlockShared<kStorage, DP, kRowGroups>::kSide;
#pragma unroll
    for (int round = 0; round < kSets / kSide; ++round) {
      if (set / kSide == round) {
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = row_group * 16 + rt * 8 + 2 * t + j;
            float top = sm.m[0][r];
#pragma unroll
            for (int o = 1; o < kSets; ++o) top = fmaxf(top, sm.m[o][r]);
            const float f = exp2_approx(st.m[rt][j] - top);
            float* row = sm.acc[set % kSide][r];
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
              // 8-bit kernels hold every four elements in the order 0, 2, 1, 3
              const int at0 = 16 * s + g, d0 = kScaled ? (at0 & ~3) | (at0 & 1) << 1 | (at0 >> 1 & 1) : at0;
              float y0 = st.o[s][rt][j] * f, y1 = st.o[s][rt][2 + j] * f;
              if (round > 0) {
                y0 += row[d0];
                y1 += row[d0 + 8];
              }
              row[d0] = y0;
              row[d0 + 8] = y1;
            }
          }
      }
      __syncthreads();
    }
    constexpr int kPerRow = kBlockThreads / kRows;
    const int r = tid / kPerRow;
    int token, head;
    row_place(a, plan, c.kv_head, c.row_block, r, token, head);
    if (token < a.q_len) {
      float top = sm.m[0][r], l = 0.f;
#pragma unroll
      for (int o = 1; o < kSets; ++o) top = fmaxf(top, sm.m[o][r]);
#pragma unroll
      for (int o = 0; o < kSets; ++o) l = fmaf(sm.l[o][r], exp2_approx(sm.m[o][r] - top), l);
      const long long tree = a.shared_tree ? 0 : static_cast<long long>(c.b) * a.q_len;
      bool empty = l == 0.f;
      if (kTree && a.depths[tree + token] < 0) empty = true;  // a padding node sees nothing
      const float inverse = 1.f / l;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + c.b * a.out_strides[0] + head * a.out_strides[1] + token * a.out_strides[2];
      float* partial = partial_row(a, plan, gridDim.x, blockIdx.x, c.tile == 0, r);
      if (!whole(c) && tid % kPerRow == 0) *reinterpret_cast<float2*>(partial) = make_float2(top, empty ? 0.f : l);
      if (kTree && sm.poison[turn] != 0) {  // drafted values that are not finite, for the rows that see them
        const int words = (a.q_len + 31) / 32;
        for (int d = 2 * (tid % kPerRow); d < a.head_dim; d += 2 * kPerRow) {
          for (int j = 0; j < a.q_len; ++j) {
            if (!(a.ancestors[(tree + token) * words + (j >> 5)] >> (j & 31) & 1u)) continue;
            const uint32_t x = *reinterpret_cast<const uint32_t*>(static_cast<const char*>(a.draft_v) +
                                                                  (c.b * a.draft_v_strides[0] + c.kv_head * a.draft_v_strides[1] + j * a.draft_v_strides[2] + d) * 2);
            if ((x & 0x7f80u) == 0x7f80u) sm.acc[0][r][d] += __uint_as_float(x << 16);
            if ((x & 0x7f800000u) == 0x7f800000u) sm.acc[0][r][d + 1] += __uint_as_float(x & 0xffff0000u);
          }
        }
      }
      const bool done = whole(c);
#pragma unroll 4
      for (int d = 2 * (tid % kPerRow); d < a.head_dim; d += 2 * kPerRow) {
        float2 y = *reinterpret_cast<const float2*>(&sm.acc[0][r][d]);
        if (kSide > 1) {
          const float2 z = *reinterpret_cast<const float2*>(&sm.acc[kSide - 1][r][d]);
          y.x += z.x;
          y.y += z.y;
        }
        if (empty) y = make_float2(0.f, 0.f);
        if (done)
          *reinterpret_cast<uint32_t*>(out + d) = empty ? 0u : pack_bf16(y.x * inverse, y.y * inverse);
        else
          *reinterpret_cast<float2*>(partial + 2 + d) = y;
      }
    }
    if (tid == 0) {
      leave_note(a, share, c, blockIdx.x, gridDim.x);
      sm.poison[turn ^ 1] = 0;
    }
    turn ^= 1;
    __syncthreads();
    if (a.head_dim < DP) {  // the sums have been over the columns behind head_dim
      for (int i = tid; i < static_cast<int>(sizeof(sm.acc) / 16); i += kBlockThreads) reinterpret_cast<uint4*>(sm.tile)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
    }
  }
}

// More than 48 KB of shared memory are opted into once per device and kernel.
struct DeviceFlags {
  static constexpr int kDevices = 64;
  std::atomic<bool> set[kDevices];
};
template <typename Kernel>
cudaError_t opt_in(Kernel* kernel, int bytes, DeviceFlags& done) {
  int device = 0;
  cudaError_t error = cudaGetDevice(&device);
  if (error != cudaSuccess) return error;
  const bool known = device >= 0 && device < DeviceFlags::kDevices;
  if (known && done.set[device].load(std::memory_order_acquire)) return cudaSuccess;
  error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (error == cudaSuccess && known) done.set[device].store(true, std::memory_order_release);
  return error;
}

template <int kStorage, int DP, int kRowGroups, bool kTree>
cudaError_t launch_shared_rows(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {
  constexpr int kBytes = static_cast<int>(sizeof(BlockShared<kStorage, DP, kRowGroups>));
  static_assert(kBytes <= 232448 / 2 - 1024, "two blocks per SM");
  static DeviceFlags done;
  const cudaError_t error = opt_in(pool_attn_shared_kernel<kStorage, DP, kRowGroups, kTree>, kBytes, done);
  if (error != cudaSuccess) return error;
  pool_attn_shared_kernel<kStorage, DP, kRowGroups, kTree><<<plan.blocks, kBlockThreads, kBytes, stream>>>(a, plan);
  return cudaGetLastError();
}

// Rows of a block: 32, 64 or 128, the largest that does not cover more rows in all than the next smaller one would (and
// whose shared memory leaves room for two blocks per SM: 64 at most over wide 8-bit rows).
inline int shared_rows_per_block(long long rows, int storage, int head_dim) {
  if (rows <= 32) return 32;
  const bool most = storage != WM_BF16 && head_dim > 64;
  return rows <= 64 || most || (rows + 127) / 128 * 128 > (rows + 63) / 64 * 64 ? 64 : 128;
}

// One translation unit per way of holding the pool.
template <int kStorage>
cudaError_t launch_shared(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream);

template <int kStorage, int DP, bool kTree>
cudaError_t launch_shared_dim(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {
  switch (plan.rows_per_block) {
    case 32: return launch_shared_rows<kStorage, DP, 2, kTree>(a, plan, stream);
    case 64: return launch_shared_rows<kStorage, DP, 4, kTree>(a, plan, stream);
  }
  if constexpr (kStorage == WM_BF16 || DP == 64) return launch_shared_rows<kStorage, DP, 8, kTree>(a, plan, stream);
  return cudaErrorInvalidValue;  // not reached: such plans have 64 rows at most
}

#define WM_POOL_SHARED_UNIT(kStorage)                                                                                             \
  template <>                                                                                                                     \
  cudaError_t launch_shared<kStorage>(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {                        \
    if (a.ancestors != nullptr)                                                                                                   \
      return a.head_dim <= 64 ? launch_shared_dim<kStorage, 64, true>(a, plan, stream) : launch_shared_dim<kStorage, 128, true>(a, plan, stream); \
    return a.head_dim <= 64 ? launch_shared_dim<kStorage, 64, false>(a, plan, stream) : launch_shared_dim<kStorage, 128, false>(a, plan, stream); \
  }

}  // namespace pool
}  // namespace wm
