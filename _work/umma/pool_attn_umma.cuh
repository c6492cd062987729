// Pool attention for bf16 queries with many rows per KV head (trees of drafted tokens, grouped heads, chunks of new tokens)
// on tcgen05: one persistent block per SM walks its share of the tiles (pool_attn_walk.cuh), 64 query rows at a time.
//
// Both products are transposed, as in pool_attn_mma.cuh: the 128 keys of a tile fill the 128 rows of the instruction and the
// query rows its columns, S^T[128 keys x 64] = K Q^T and O^T[head_dim x 64] += V^T P^T, so a tile costs the same few
// instructions for 17 rows as for 64, and a thread of the soft-max owns a key: its scale, its value's scale and its
// visibility are scalars.  What is uncommon in that layout is the row maximum, which runs across the 128 threads: rows keep a
// reference that moves only when a score exceeds it by 2^8, and the common tile needs one vote of the 128 threads.
//
//   warps 0-7   soft-max, two groups of 128 threads on alternate tiles, each with its own references, sums and output
//               accumulator (a tile takes a group about 2 000 cycles from its scores to its weights, most of it latency, and
//               HBM brings a tile of 64-element bf16 rows every 1 430): a tile's scores from tensor memory, weights to
//               shared memory as bf16 (the B operand of the value product, 64 rows = one 128-byte swizzle line per key);
//               at a segment's end the two meet and write the output
//   warps 8-11  loaders: pool rows to swizzled bf16 tiles.  bf16 rows by asynchronous 16-byte copies straight into
//               place; 8-bit rows by the same copies into a private corner of shared memory per thread, from where the
//               thread turns its own codes into bf16 (exact) and stores them; rows that are not visible as zeros
//   warps 12-13 issue the products, one the scores, one the values: an issuing thread is busy for as long as the pipe
//               works on what it issued
//
// Every wait on a barrier is bounded (pool_wait): when one gives up, the block's abort flag ends all other waits of the
// block at once, the roles run their loops to the end on whatever is there, nothing is skipped that another role counts
// on, and the status word says which wait it was.  Every barrier is closed into a loop: its producers' next phase depends
// on its consumers having seen the last.
#pragma once

#include "pool_attn_mma.cuh"
#include "sm100_ptx.cuh"

namespace wm {
namespace pool {

constexpr int kUmmaRows = 64;
constexpr int kSoftmaxThreads = 256;
constexpr int kLoadWarps = 4, kLoaders = kLoadWarps * 32;
constexpr int kUmmaThreads = kSoftmaxThreads + kLoaders + 64;
constexpr int kSumSlots = 8;  // tiles whose scales and visibility are held

template <int kStorage, int DP>
struct Umma {
  static constexpr int kBytes = kStorage == WM_BF16 ? 2 : 1;
  static constexpr int kSub = DP / 64;                    // a tile is kSub sub-tiles of 64 columns, 128 keys x 128 bytes each
  static constexpr int kTileBytes = kSub * 16384;
  static constexpr int kStages = DP == 64 ? (kStorage == WM_BF16 ? 5 : 3) : 2;
  static constexpr int kRaw = kStorage == WM_BF16 ? 0 : (DP == 64 ? 3 : 1);  // tiles of codes in flight
  static constexpr int kQueries = DP == 64 ? 2 : 1;       // query tiles held
  static constexpr int kChunks = DP * kBytes / 16;        // 16-byte pieces of a row
  static constexpr int kPasses = 128 * kChunks / kLoaders;  // pieces of a K (or V) tile per loader thread
};

template <int kStorage, int DP>
struct UmmaShared {
  using C = Umma<kStorage, DP>;
  unsigned char k[C::kStages][2][C::kTileBytes];  // [stage][K, V]
  unsigned char p[2][16384];                      // weights, per group; at a segment's end 32 rows of the group's output, [32][DP] floats
  unsigned char q[C::kQueries][C::kSub * 8192];
  uint4 raw[C::kRaw > 0 ? C::kRaw : 1][2][C::kRaw > 0 ? C::kPasses : 1][C::kRaw > 0 ? kLoaders : 1];
  float scale[kSumSlots][2][128];                 // key and value scales of a tile's rows
  unsigned char seen[kSumSlots][128];             // key_mask of a tile's rows
  uint32_t bits[8][kUmmaRows];                    // ancestor words of the rows for one warp's 32 drafted tokens
  float reference[2][kUmmaRows];                  // minus the rows' references, per group
  float moved[2][kUmmaRows];                      // what a reference that moved multiplies the row's sums with
  float top[8][32];
  float sum[8][kUmmaRows];
  uint64_t full[C::kStages], empty[C::kStages], s_full[2], s_empty[2], p_full[2], p_empty[2], q_empty[2], o_empty[2], done[2];
  uint32_t tmem;
  int abort_flag;
  int poison[8];  // a piece's drafted values hold an infinity or NaN
  int* status;
};

template <class Shared>
__device__ __forceinline__ void pool_wait(Shared& sm, uint64_t* bar, uint32_t parity, int code) {
  if (ptx::mbar_try_wait(bar, parity)) return;
  const long long begin = clock64();
  for (uint32_t spin = 0;; ++spin) {
    if (ptx::mbar_try_wait(bar, parity)) return;
    if ((spin & 3u) == 3u) {
      if (*reinterpret_cast<volatile int*>(&sm.abort_flag)) return;
      if (clock64() - begin > 400000000ll) break;  // 0.2 s
    }
  }
  atomicCAS(sm.status, 0, code | static_cast<int>((blockIdx.x & 0x7fffffu) << 8));
  atomicExch(&sm.abort_flag, 1);
}

// The tiles of a share, one after another.
struct Walk {
  Share share;
  Piece c;
  int at, tile, piece;  // `at`: first unit behind the current piece
  bool valid, has_draft;

  __device__ void start(const wm_pool_attn_args& a, const Plan& p) {
    share = find_share(a, p, blockIdx.x, gridDim.x);
    has_draft = p.draft_tiles > 0;
    at = share.begin;
    piece = -1;
    valid = true;
    c.stop = tile = 0;
    next(a, p);
  }
  __device__ void next(const wm_pool_attn_args& a, const Plan& p) {
    if (++tile < c.stop) return;
    do {
      if (at >= share.end) {
        valid = false;
        return;
      }
      c = next_piece(a, p, at, share.end, share.b, share.b_begin);
      at = c.end;
    } while (c.tile >= c.stop);
    tile = c.tile;
    ++piece;
  }
  __device__ bool first() const { return tile == c.tile; }
  __device__ bool last() const { return tile + 1 == c.stop; }
  __device__ bool draft() const { return has_draft && tile >= c.past_tiles; }
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16u : 0u) : "memory");
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
// 16-byte piece `piece` (8 bf16 elements) of row `row` of a tile of 128-byte swizzled rows, `sub_bytes` per 64 columns
__device__ __forceinline__ uint32_t swizzled(int row, int piece, int sub_bytes) {
  return (piece >> 3) * sub_bytes + row * 128 + (((piece & 7) ^ (row & 7)) << 4);
}
// Elements 4i .. 4i + 3 in the order 0, 2, 1, 3 (how a word of codes comes apart; the queries and drafted rows follow)
__device__ __forceinline__ uint4 permuted(const uint4& x) {
  return make_uint4(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632), __byte_perm(x.z, x.w, 0x5410), __byte_perm(x.z, x.w, 0x7632));
}
__device__ __forceinline__ uint32_t finite_halves(uint32_t x, bool& special) {
  if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u, special = true;
  if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu, special = true;
  return x;
}

// ---------------------------------------------------------------- loaders
template <int kValue>
struct Count {
  static constexpr int value = kValue;
};

template <int kStorage, int DP>
struct Loader {
  using C = Umma<kStorage, DP>;
  static constexpr int kRaw = C::kRaw > 0 ? C::kRaw : 1;
  UmmaShared<kStorage, DP>& sm;
  const wm_pool_attn_args& a;
  const Plan& plan;
  const int tid = threadIdx.x - kSoftmaxThreads;

  // Queries of the walk's piece, rows that do not exist as zeros.
  __device__ void load_queries(const Walk& w) {
    const int buffer = w.piece % C::kQueries;
    const uint32_t base = ptx::smem_u32(sm.q[buffer]);
    constexpr int kPieces = DP / 8;
#pragma unroll 2
    for (int i = tid; i < kUmmaRows * kPieces; i += kLoaders) {
      const int row = i / kPieces, piece = i % kPieces;
      int token, head;
      row_place(a, plan, w.c.kv_head, w.c.row_block, row, token, head);
      uint4 x = make_uint4(0, 0, 0, 0);
      if (token < a.q_len && piece * 8 < a.head_dim)
        x = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.q) + (w.c.b * a.q_strides[0] + head * a.q_strides[1] + token * a.q_strides[2] + piece * 8) * 2);
      if (kStorage != WM_BF16) x = permuted(x);
      st_shared_16(base + swizzled(row, piece, 8192), x);
    }
  }

  // A tile of drafted tokens, by plain loads: padding nodes as zeros, and values that are not finite as zeros with a note
  // (an infinity or NaN must reach the rows that see it, and a product would carry it to all).
  __device__ void load_draft(const Walk& w, int stage) {
    const long long tree = a.shared_tree ? 0 : static_cast<long long>(w.c.b) * a.q_len;
    constexpr int kPieces = DP / 8;
    const uint32_t to[2] = {ptx::smem_u32(sm.k[stage][0]), ptx::smem_u32(sm.k[stage][1])};
    bool special = false;
#pragma unroll 1
    for (int i = tid; i < 2 * 128 * kPieces; i += kLoaders) {
      const int value = i / (128 * kPieces), row = i / kPieces % 128, piece = i % kPieces;
      const int j = (w.tile - w.c.past_tiles) * kTileKeys + row;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (j < a.q_len && piece * 8 < a.head_dim && a.depths[tree + j] >= 0) {
        const int64_t* strides = value ? a.draft_v_strides : a.draft_k_strides;
        x = *reinterpret_cast<const uint4*>(static_cast<const char*>(value ? a.draft_v : a.draft_k) +
                                            (w.c.b * strides[0] + w.c.kv_head * strides[1] + j * strides[2] + piece * 8) * 2);
      }
      if (value) x = make_uint4(finite_halves(x.x, special), finite_halves(x.y, special), finite_halves(x.z, special), finite_halves(x.w, special));
      if (kStorage != WM_BF16) x = permuted(x);
      st_shared_16((value ? to[1] : to[0]) + swizzled(row, piece, 16384), x);
    }
    if (special) sm.poison[w.piece & 7] = 1;
  }

  // Where this thread's part of the walk's tile lies: set at the start of a piece, moved on tile by tile.
  struct Source {
    const char *k, *v;
    const float *k_scale, *v_scale;
    const uint8_t* mask;
    uint32_t k_pass, v_pass;  // bytes between the rows of two passes
    bool inside;              // this thread's 16 bytes of a row lie in front of head_dim
  };
  __device__ void set_source(Source& s, const Walk& w) const {
    const int row = tid / C::kChunks, piece = tid % C::kChunks;
    const long long j = static_cast<long long>(w.tile) * kTileKeys + row;
    static_assert(kLoaders == kTileKeys, "a thread fetches one row's scales");
    s.k = static_cast<const char*>(a.k) + (w.c.b * a.k_strides[0] + w.c.kv_head * a.k_strides[1] + j * a.k_strides[2]) * C::kBytes + piece * 16;
    s.v = static_cast<const char*>(a.v) + (w.c.b * a.v_strides[0] + w.c.kv_head * a.v_strides[1] + j * a.v_strides[2]) * C::kBytes + piece * 16;
    s.k_pass = static_cast<uint32_t>(kLoaders / C::kChunks * a.k_strides[2]) * C::kBytes;
    s.v_pass = static_cast<uint32_t>(kLoaders / C::kChunks * a.v_strides[2]) * C::kBytes;
    s.inside = piece * 16 < a.head_dim * C::kBytes;
    s.mask = a.key_mask != nullptr ? a.key_mask + static_cast<long long>(w.c.b) * a.k_len : nullptr;
    if (kStorage != WM_BF16) {
      const long long at = static_cast<long long>(w.tile) * kTileKeys + tid;
      s.k_scale = a.k_scales + w.c.b * a.k_scale_strides[0] + w.c.kv_head * a.k_scale_strides[1] + at * a.k_scale_strides[2];
      s.v_scale = a.v_scales + w.c.b * a.v_scale_strides[0] + w.c.kv_head * a.v_scale_strides[1] + at * a.v_scale_strides[2];
    }
  }
  __device__ void move_source(Source& s) const {
    s.k += kTileKeys * a.k_strides[2] * C::kBytes;
    s.v += kTileKeys * a.v_strides[2] * C::kBytes;
    if (kStorage != WM_BF16) {
      s.k_scale += kTileKeys * a.k_scale_strides[2];
      s.v_scale += kTileKeys * a.v_scale_strides[2];
    }
  }

  // Asks for this thread's part of the keys (v = 0) or values of a tile: straight into the stage (bf16) or into its raw
  // corner (8 bits), and for the tile's scales and mask.
  __device__ void ask(Source& s, const Walk& w, int n, int v) {
    if (v == 0) {
      if (w.first())
        set_source(s, w);
      else
        move_source(s);
    }
    const int j0 = w.tile * kTileKeys, slot = n % kSumSlots, row0 = tid / C::kChunks, piece = tid % C::kChunks;
    constexpr int kStep = kLoaders / C::kChunks;  // rows of a pass: a multiple of 8, so the swizzle of a thread's rows is one
    const uint32_t to = kStorage == WM_BF16 ? ptx::smem_u32(sm.k[n % C::kStages][v]) + swizzled(row0, piece, 16384)
                                            : ptx::smem_u32(&sm.raw[n % kRaw][v][0][kStorage == WM_BF16 ? 0 : tid]);
    constexpr int kTo = kStorage == WM_BF16 ? kStep * 128 : kLoaders * 16;
    const char* src = v ? s.v : s.k;
    const uint32_t pass = v ? s.v_pass : s.k_pass;
    if (s.inside) {  // columns behind head_dim stay as they were set up: zeros
      if (s.mask == nullptr && j0 + kTileKeys <= w.c.slots) {
#pragma unroll
        for (int i = 0; i < C::kPasses; ++i) cp_async_16(to + i * kTo, src + i * pass, true);
      } else {
        bool live[C::kPasses];
#pragma unroll
        for (int i = 0; i < C::kPasses; ++i) {
          const int j = j0 + row0 + i * kStep;
          live[i] = j < w.c.slots && (s.mask == nullptr || s.mask[j] != 0);
        }
#pragma unroll
        for (int i = 0; i < C::kPasses; ++i) cp_async_16(to + i * kTo, live[i] ? src + i * pass : static_cast<const char*>(a.k), live[i]);
      }
    }
    const bool there = j0 + tid < w.c.slots;
    if (kStorage != WM_BF16) ptx::cp_async_4(&sm.scale[slot][v][tid], there ? (v ? s.v_scale : s.k_scale) : a.k_scales, there);
    if (v == 0 && s.mask != nullptr) sm.seen[slot][tid] = there ? s.mask[j0 + tid] : 0;
  }

  // Turns this thread's codes of the keys (v = 0) or values into bf16, in the tile's stage.
  __device__ void convert(const uint4 (&raw)[C::kPasses], int n, int v) {
    const int row0 = tid / C::kChunks, piece = tid % C::kChunks;
    if (piece * 16 >= a.head_dim) return;
    const uint32_t to = ptx::smem_u32(sm.k[n % C::kStages][v]);
    const uint32_t first = to + swizzled(row0, 2 * piece, 16384), second = to + swizzled(row0, 2 * piece + 1, 16384);
    constexpr int kTo = kLoaders / C::kChunks * 128;
#pragma unroll
    for (int i = 0; i < C::kPasses; ++i) {
      const uint4 x = raw[i];
      st_shared_16(first + i * kTo, make_uint4(Codes<kStorage>::even(x.x), Codes<kStorage>::odd(x.x), Codes<kStorage>::even(x.y), Codes<kStorage>::odd(x.y)));
      st_shared_16(second + i * kTo, make_uint4(Codes<kStorage>::even(x.z), Codes<kStorage>::odd(x.z), Codes<kStorage>::even(x.w), Codes<kStorage>::odd(x.w)));
    }
  }

  __device__ void arrive(int n) {
    ptx::fence_async_shared();
    __syncwarp();
    if ((tid & 31) == 0) ptx::mbar_arrive(&sm.full[n % C::kStages]);
  }
  // The stage of tile n, the query buffer of the walk's piece are free again.  `flush` is called by a warp that would have to
  // wait: what it waits for may depend on tiles that it has not reported yet.  It reports them as they land, until the
  // question it is given says that the wait is over.
  template <class Flush>
  __device__ void wait_free(uint64_t* bar, uint32_t parity, int code, const Flush& flush) {
    const auto free = [&] { return __all_sync(0xffffffffu, ptx::mbar_test_wait(bar, parity)) != 0; };
    if (!free()) {
      flush(free);
      pool_wait(sm, bar, parity, code);
    }
  }
  template <class Flush>
  __device__ void wait_empty(int n, const Flush& flush) {
    if (n >= C::kStages) wait_free(&sm.empty[n % C::kStages], ((n / C::kStages) & 1) ^ 1, 202, flush);
  }
  template <class Flush>
  __device__ void wait_queries(const Walk& w, const Flush& flush) {
    if (w.piece >= C::kQueries) wait_free(&sm.q_empty[w.piece % C::kQueries], ((w.piece / C::kQueries) & 1) ^ 1, 201, flush);
  }

  __device__ void run() {
    Walk w;
    w.start(a, plan);
    int n = 0;
    if (kStorage == WM_BF16) {
      // a tile is reported once it has landed: kAhead tiles later, or when there is nothing to do but wait
      constexpr int kAhead = C::kStages - 1;
      int reported = 0;
      Source source;
      const auto landed = [&](auto pending) {  // all but the `pending` newest tiles
        cp_async_wait<decltype(pending)::value>();
        for (; reported < n - decltype(pending)::value; ++reported) arrive(reported);
      };
      const auto flush = [&](const auto& free) {
        if constexpr (kAhead > 3) {
          landed(Count<3>());
          if (free()) return;
        }
        if constexpr (kAhead > 2) {
          landed(Count<2>());
          if (free()) return;
        }
        if constexpr (kAhead > 1) {
          landed(Count<1>());
          if (free()) return;
        }
        landed(Count<0>());
      };
      for (; w.valid; ++n, w.next(a, plan)) {
        wait_empty(n, flush);
        if (w.first()) {
          wait_queries(w, flush);
          load_queries(w);
        }
        if (w.draft()) {
          load_draft(w, n % C::kStages);
        } else {
          ask(source, w, n, 0);
          ask(source, w, n, 1);
        }
        ptx::cp_async_commit();
        landed(Count<kAhead>());
      }
      landed(Count<0>());
    } else {
      // keys and values of a tile are asked for in groups of their own, kRaw tiles ahead of their turn
      Walk ahead = w;
      Source source;
      int m = 0;
      const auto ask_next = [&](int v) {
        if (ahead.valid && !ahead.draft()) ask(source, ahead, m, v);
        ptx::cp_async_commit();
        if (v == 1 && ahead.valid) {
          ++m;
          ahead.next(a, plan);
        }
      };
#pragma unroll
      for (int i = 0; i < kRaw; ++i) {
        ask_next(0);
        ask_next(1);
      }
      for (; w.valid; ++n, w.next(a, plan)) {
        const auto nothing = [](const auto&) {};
        wait_empty(n, nothing);
        if (w.first()) {
          wait_queries(w, nothing);
          load_queries(w);
        }
        if (w.draft()) load_draft(w, n % C::kStages);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          cp_async_wait<2 * kRaw - 1>();  // this tile's codes have landed
          uint4 raw[C::kPasses];
          if (!w.draft()) {
#pragma unroll
            for (int i = 0; i < C::kPasses; ++i) raw[i] = ld_shared_16(ptx::smem_u32(&sm.raw[n % kRaw][v][kStorage == WM_BF16 ? 0 : i][kStorage == WM_BF16 ? 0 : tid]));
          }
          const bool draft = w.draft();
          ask_next(v);
          if (!draft) convert(raw, n, v);
        }
        arrive(n);
      }
      cp_async_wait<0>();
    }
  }
};

// ---------------------------------------------------------------- products
// Tensor memory: scores of the two groups' tiles in columns [0, 64) and [64, 128), their outputs in [128, 192) and [192, 256).
constexpr uint32_t kUmmaOutput = 128, kUmmaColumns = 256;

// One lane of a warp each, after the warp has found its share together.
template <int kStorage, int DP>
__device__ void issue_scores(UmmaShared<kStorage, DP>& sm, const wm_pool_attn_args& a, const Plan& plan, Walk& w) {
  using C = Umma<kStorage, DP>;
  constexpr uint32_t idesc = ptx::make_idesc_bf16(128, kUmmaRows, 0, 0);  // K Q^T, head_dim contiguous in both
  const uint32_t tmem = sm.tmem;
  for (int n = 0; w.valid; ++n, w.next(a, plan)) {
    const int stage = n % C::kStages;
    if (n >= 2) pool_wait(sm, &sm.s_empty[n & 1], ((n >> 1) & 1) ^ 1, 203);
    pool_wait(sm, &sm.full[stage], (n / C::kStages) & 1, 204);
    ptx::tc_fence_after();
    const uint64_t k = ptx::make_smem_desc_sw128(ptx::smem_u32(sm.k[stage][0]), 16, 1024);
    const uint64_t q = ptx::make_smem_desc_sw128(ptx::smem_u32(sm.q[w.piece % C::kQueries]), 16, 1024);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s)
      ptx::mma_bf16_ss(tmem + (n & 1) * kUmmaRows, ptx::desc_advance(k, (s >> 2) * 16384 + (s & 3) * 32), ptx::desc_advance(q, (s >> 2) * 8192 + (s & 3) * 32),
                       idesc, s > 0);
    ptx::mma_commit(&sm.s_full[n & 1]);
    if (w.last()) ptx::mma_commit(&sm.q_empty[w.piece % C::kQueries]);
  }
  ptx::mma_commit(&sm.done[0]);
  pool_wait(sm, &sm.done[0], 0, 209);  // nothing is in flight when the block ends
}

template <int kStorage, int DP>
__device__ void issue_values(UmmaShared<kStorage, DP>& sm, const wm_pool_attn_args& a, const Plan& plan, Walk& w) {
  using C = Umma<kStorage, DP>;
  constexpr uint32_t idesc = ptx::make_idesc_bf16(128, kUmmaRows, 1, 1);  // V^T P^T, keys strided in both
  const uint32_t tmem = sm.tmem;
  int pieces[2] = {0, 0};  // segments that each group has had a tile of
  for (int n = 0; w.valid; ++n, w.next(a, plan)) {
    const int stage = n % C::kStages, group = n & 1;
    const bool first = w.tile - w.c.tile < 2;  // the group's first tile of the piece
    pool_wait(sm, &sm.full[stage], (n / C::kStages) & 1, 210);
    pool_wait(sm, &sm.p_full[group], (n >> 1) & 1, 211);
    if (first) {
      const int before = group ? pieces[1] : pieces[0];
      if (before > 0) pool_wait(sm, &sm.o_empty[group], (before & 1) ^ 1, 212);
      if (group)
        ++pieces[1];
      else
        ++pieces[0];
    }
    ptx::tc_fence_after();
    // head_dim of 64: the instruction's upper 64 rows read what lies behind the tile (shared memory of this block); nobody
    // reads the lanes they end up in
    const uint64_t v = ptx::make_smem_desc_sw128(ptx::smem_u32(sm.k[stage][1]), 16384, 1024);
    const uint64_t p = ptx::make_smem_desc_sw128(ptx::smem_u32(sm.p[group]), 16384, 1024);
#pragma unroll
    for (int s = 0; s < 8; ++s)
      ptx::mma_bf16_ss(tmem + kUmmaOutput + group * kUmmaRows, ptx::desc_advance(v, s * 2048), ptx::desc_advance(p, s * 2048), idesc, !first || s > 0);
    ptx::mma_commit(&sm.p_empty[group]);
    ptx::mma_commit(&sm.empty[stage]);
  }
  ptx::mma_commit(&sm.done[1]);
  pool_wait(sm, &sm.done[1], 0, 213);
}

// ---------------------------------------------------------------- soft-max
__device__ __forceinline__ void group_barrier(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
__device__ __forceinline__ void both_groups_barrier() { asm volatile("bar.sync 3, 256;" ::: "memory"); }
__device__ __forceinline__ bool group_any(int group, bool x) {
  uint32_t y;
  asm volatile("{.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbar.red.or.pred q, %2, 128, p;\nselp.b32 %0, 1, 0, q;}"
               : "=r"(y)
               : "r"(static_cast<uint32_t>(x)), "r"(1 + group)
               : "memory");
  return y != 0;
}
// x[i] over the 32 lanes for every i; lane i keeps the result of x[i].
template <bool kMax>
__device__ __forceinline__ float across_lanes(float (&x)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = lane & o ? x[i] : x[i + o], keep = lane & o ? x[i + o] : x[i];
      const float got = __shfl_xor_sync(0xffffffffu, give, o);
      x[i] = kMax ? fmaxf(keep, got) : keep + got;
    }
  return x[0];
}

// Chunks of 32 rows that exist (kRowChunks 1 or 2) are what the soft-max works on; columns of the others hold what was there.
template <int kStorage, int DP, bool kTree, int kRowChunks>
__device__ void softmax(UmmaShared<kStorage, DP>& sm, const wm_pool_attn_args& a, const Plan& plan) {
  constexpr bool kScaled = kStorage != WM_BF16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = warp >> 2, tid = threadIdx.x & 127;  // tid: the key of a tile
  const uint32_t tmem = sm.tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
  const uint32_t output = tmem + kUmmaOutput + group * kUmmaRows;
  float* const reference = sm.reference[group];
  float* const moved = sm.moved[group];
  const float factor = a.scale * kLog2e;
  Walk w;
  w.start(a, plan);
  float l[kRowChunks][32];
  for (int n = 0; w.valid; ++n, w.next(a, plan)) {
    if (w.first()) {
#pragma unroll
      for (int h = 0; h < kRowChunks; ++h)
#pragma unroll
        for (int i = 0; i < 32; ++i) l[h][i] = 0.f;
      if (tid < kUmmaRows) reference[tid] = -kNoReference;
      group_barrier(group);
    }
    if ((n & 1) == group) {
      const bool first = w.tile - w.c.tile < 2, draft = kTree && w.draft();
      if (draft) {  // this warp's 32 drafted tokens are one word of every row
        const int words = (a.q_len + 31) / 32, word = (w.tile - w.c.past_tiles) * 4 + (warp & 3);
        const long long tree = a.shared_tree ? 0 : static_cast<long long>(w.c.b) * a.q_len;
#pragma unroll
        for (int h = 0; h < kRowChunks; ++h) {
          int token, head;
          row_place(a, plan, w.c.kv_head, w.c.row_block, h * 32 + lane, token, head);
          sm.bits[warp][h * 32 + lane] = token < a.q_len && word < words ? a.ancestors[(tree + token) * words + word] : 0u;
        }
        __syncwarp();
      }
      pool_wait(sm, &sm.s_full[group], (n >> 1) & 1, 205);
      ptx::tc_fence_after();
      bool seen = true;
      float f = factor, value_scale = 1.f;
      if (!draft) {
        seen = w.tile * kTileKeys + tid < w.c.slots;
        if (a.key_mask != nullptr) seen = seen && sm.seen[n % kSumSlots][tid] != 0;
        if (kScaled) {
          f = seen ? factor * sm.scale[n % kSumSlots][0][tid] : 0.f;
          value_scale = seen ? sm.scale[n % kSumSlots][1][tid] : 0.f;
        }
      }
      const bool all = !draft && __all_sync(0xffffffffu, seen);
      const uint32_t p_row = ptx::smem_u32(sm.p[group]) + tid * 128;
#pragma unroll
      for (int h = 0; h < kRowChunks; ++h) {
        uint32_t raw[32];
        const uint32_t at = tmem + group * kUmmaRows + 32 * h;
        ptx::tmem_ld32(at, raw);
        ptx::tmem_wait_ld();
        float x[32];
        const auto mask = [&] {
          if (draft) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const uint4 bits = *reinterpret_cast<const uint4*>(&sm.bits[warp][32 * h + i]);
              if (!(bits.x >> lane & 1u)) x[i] = -INFINITY;
              if (!(bits.y >> lane & 1u)) x[i + 1] = -INFINITY;
              if (!(bits.z >> lane & 1u)) x[i + 2] = -INFINITY;
              if (!(bits.w >> lane & 1u)) x[i + 3] = -INFINITY;
            }
          } else if (!all) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!seen) x[i] = -INFINITY;
          }
        };
        const auto against_reference = [&] {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 ref = *reinterpret_cast<const float4*>(&reference[32 * h + i]);
            x[i] = fmaf(__uint_as_float(raw[i]), f, ref.x);
            x[i + 1] = fmaf(__uint_as_float(raw[i + 1]), f, ref.y);
            x[i + 2] = fmaf(__uint_as_float(raw[i + 2]), f, ref.z);
            x[i + 3] = fmaf(__uint_as_float(raw[i + 3]), f, ref.w);
          }
          mask();
        };
        against_reference();
        float part[4] = {x[0], x[1], x[2], x[3]};  // four short chains
#pragma unroll
        for (int i = 4; i < 32; i += 4)
#pragma unroll
          for (int e = 0; e < 4; ++e) part[e] = fmaxf(part[e], x[i + e]);
        if (group_any(group, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) > kReferenceSlack)) {
          // some row's reference has to move: the rows' true maxima over the tile, from the scores once more
          ptx::tmem_ld32(at, raw);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(raw[i]) * f;
          mask();
          sm.top[warp][lane] = across_lanes<true>(x);
          group_barrier(group);
          if ((warp & 3) == 0) {
            const float old = -reference[32 * h + lane];
            const float now = fmaxf(fmaxf(fmaxf(sm.top[warp][lane], sm.top[warp + 1][lane]), fmaxf(sm.top[warp + 2][lane], sm.top[warp + 3][lane])), old);
            moved[32 * h + lane] = exp2_approx(old - now);
            reference[32 * h + lane] = -now;
          }
          group_barrier(group);
#pragma unroll
          for (int i = 0; i < 32; ++i) l[h][i] *= moved[32 * h + i];
          if (!first) {  // the group's output so far: its last product has to be complete
            pool_wait(sm, &sm.p_empty[group], ((n >> 1) & 1) ^ 1, 206);
            ptx::tc_fence_after();
            ptx::tmem_ld32(output + 32 * h, raw);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) raw[i] = __float_as_uint(__uint_as_float(raw[i]) * moved[32 * h + i]);
            ptx::tmem_st32(output + 32 * h, raw);
            ptx::tmem_wait_st();
          }
          ptx::tmem_ld32(at, raw);
          ptx::tmem_wait_ld();
          against_reference();
        }
        if (h == kRowChunks - 1) {  // the scores have been read
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&sm.s_empty[group]);
        }
        if (h == 0 && n >= 2) pool_wait(sm, &sm.p_empty[group], ((n >> 1) & 1) ^ 1, 207);
        uint32_t pack[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float p0 = exp2_approx(x[i]), p1 = exp2_approx(x[i + 1]);
          if (kScaled) {
            l[h][i] += p0, l[h][i + 1] += p1;
            p0 *= value_scale, p1 *= value_scale;
          }
          pack[i / 2] = pack_bf16(p0, p1);
          if (!kScaled) ptx::add_bf16_halves(pack[i / 2], l[h][i], l[h][i + 1]);  // the sum takes the weights as they are rounded
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st_shared_16(p_row + (((4 * h + i) ^ (tid & 7)) << 4), make_uint4(pack[4 * i], pack[4 * i + 1], pack[4 * i + 2], pack[4 * i + 3]));
      }
      ptx::fence_async_shared();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&sm.p_full[group]);
    }

    if (w.last()) {
      const Piece& c = w.c;
      // the group's last tile of the piece; a piece of one tile leaves the other group without any
      const int newest = (n & 1) == group ? n : n - 1;
      const bool any = newest - (n - (w.tile - c.tile)) >= 0;
#pragma unroll
      for (int h = 0; h < kRowChunks; ++h) sm.sum[warp][32 * h + lane] = across_lanes<false>(l[h]);
      if (any) {
        pool_wait(sm, &sm.p_empty[group], (newest >> 1) & 1, 208);
        ptx::tc_fence_after();
      }
      const long long tree = a.shared_tree ? 0 : static_cast<long long>(c.b) * a.q_len;
#pragma unroll 1
      for (int h = 0; h < kRowChunks; ++h) {
        // 32 rows of either group's output through its weights' place
        const int lane_d = (warp & 3) * 32 + lane, d_of = kScaled ? (lane_d & ~3) | ((lane_d & 1) << 1) | ((lane_d >> 1) & 1) : lane_d;
        float* mine = reinterpret_cast<float*>(sm.p[group]);
        if (any && lane_d < DP) {
          uint32_t raw[32];
          ptx::tmem_ld32(output + 32 * h, raw);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) mine[i * DP + d_of] = __uint_as_float(raw[i]);
        } else {
          for (int i = 0; i < 32 && lane_d < DP; ++i) mine[i * DP + d_of] = 0.f;
        }
        if (any && h == kRowChunks - 1) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&sm.o_empty[group]);
        }
        both_groups_barrier();
        const bool poisoned = kTree && sm.poison[w.piece & 7] != 0;  // (the group of the last tile has seen it arrive)
#pragma unroll 1
        for (int i = warp; i < 32; i += 8) {
          const int r = 32 * h + i;
          int token, head;
          row_place(a, plan, c.kv_head, c.row_block, r, token, head);
          if (token >= a.q_len) break;
          const float ref0 = -sm.reference[0][r], ref1 = -sm.reference[1][r], top = fmaxf(ref0, ref1);
          const float f0 = exp2_approx(ref0 - top), f1 = exp2_approx(ref1 - top);
          const float sum = (sm.sum[0][r] + sm.sum[1][r] + sm.sum[2][r] + sm.sum[3][r]) * f0 + (sm.sum[4][r] + sm.sum[5][r] + sm.sum[6][r] + sm.sum[7][r]) * f1;
          bool empty = sum == 0.f;
          if (kTree && a.depths[tree + token] < 0) empty = true;  // a padding node sees nothing
          const float inverse = 1.f / sum;
          float* partial = partial_row(a, plan, gridDim.x, blockIdx.x, c.tile == 0, r);
          if (!whole(c) && lane == 0) *reinterpret_cast<float2*>(partial) = make_float2(top, empty ? 0.f : sum);
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + c.b * a.out_strides[0] + head * a.out_strides[1] + token * a.out_strides[2];
#pragma unroll
          for (int d = 2 * lane; d < DP; d += 64) {
            if (d >= a.head_dim) break;
            const float2 y0 = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(sm.p[0]) + i * DP + d);
            const float2 y1 = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(sm.p[1]) + i * DP + d);
            float2 y = make_float2(y0.x * f0 + y1.x * f1, y0.y * f0 + y1.y * f1);
            if (poisoned) {  // drafted values that are not finite, for the rows that see them
              const int words = (a.q_len + 31) / 32;
              for (int j = 0; j < a.q_len; ++j) {
                if (!(a.ancestors[(tree + token) * words + (j >> 5)] >> (j & 31) & 1u)) continue;
                const uint32_t x = *reinterpret_cast<const uint32_t*>(static_cast<const char*>(a.draft_v) +
                                                                      (c.b * a.draft_v_strides[0] + c.kv_head * a.draft_v_strides[1] + j * a.draft_v_strides[2] + d) * 2);
                if ((x & 0x7f80u) == 0x7f80u) y.x += __uint_as_float(x << 16);
                if ((x & 0x7f800000u) == 0x7f800000u) y.y += __uint_as_float(x & 0xffff0000u);
              }
            }
            if (empty) y = make_float2(0.f, 0.f);
            if (whole(c))
              *reinterpret_cast<uint32_t*>(out + d) = empty ? 0u : pack_bf16(y.x * inverse, y.y * inverse);
            else
              *reinterpret_cast<float2*>(partial + 2 + d) = y;
          }
        }
        both_groups_barrier();  // the rows make way for the next ones, for weights, the references for the next segment's
      }
      if (threadIdx.x == 0) {
        leave_note(a, w.share, c, blockIdx.x, gridDim.x);
        if (kTree) sm.poison[w.piece & 7] = 0;
      }
    }
  }
}

template <int kStorage, int DP, bool kTree>
__global__ void __launch_bounds__(kUmmaThreads, 1) pool_attn_umma_kernel(const wm_pool_attn_args a, const Plan plan, int* status) {
  using C = Umma<kStorage, DP>;
  extern __shared__ unsigned char smem_raw[];
  UmmaShared<kStorage, DP>& sm = *reinterpret_cast<UmmaShared<kStorage, DP>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      ptx::mbar_init(&sm.full[i], kLoadWarps);
      ptx::mbar_init(&sm.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&sm.s_full[i], 1);
      ptx::mbar_init(&sm.s_empty[i], 4);
      ptx::mbar_init(&sm.p_full[i], 4);
      ptx::mbar_init(&sm.p_empty[i], 1);
      ptx::mbar_init(&sm.q_empty[i], 1);
      ptx::mbar_init(&sm.o_empty[i], 4);
      ptx::mbar_init(&sm.done[i], 1);
    }
    ptx::mbar_fence_init();
    sm.abort_flag = 0;
    sm.status = status;
    for (int i = 0; i < 8; ++i) sm.poison[i] = 0;
    note_of(a, blockIdx.x)->last = -1;
  }
  // tiles and weights start as zeros: columns behind head_dim and rows that do not exist must not hold NaN
  for (int i = tid; i < static_cast<int>(sizeof(sm.k) / 16); i += kUmmaThreads) reinterpret_cast<uint4*>(sm.k)[i] = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < static_cast<int>(sizeof(sm.p) / 16); i += kUmmaThreads) reinterpret_cast<uint4*>(sm.p)[i] = make_uint4(0, 0, 0, 0);
  ptx::fence_async_shared();
  if (warp == 12) {
    ptx::tmem_alloc(&sm.tmem, kUmmaColumns);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // 448 threads were launched with 128 registers each: 256 x 144 + 128 x 96 + 64 x 128 is the same sum
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    if (plan.group * static_cast<long long>(a.q_len) <= 32)
      softmax<kStorage, DP, kTree, 1>(sm, a, plan);
    else
      softmax<kStorage, DP, kTree, 2>(sm, a, plan);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    Loader<kStorage, DP> loader{sm, a, plan};
    loader.run();
  } else {
    Walk w;
    w.start(a, plan);
    if ((tid & 31) == 0) {
      if (warp == 12)
        issue_scores<kStorage, DP>(sm, a, plan, w);
      else
        issue_values<kStorage, DP>(sm, a, plan, w);
    }
    __syncwarp();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 12) ptx::tmem_dealloc(sm.tmem, kUmmaColumns);
}

template <int kStorage, int DP, bool kTree>
cudaError_t launch_umma_dim(const wm_pool_attn_args& a, const Plan& plan, int* status, cudaStream_t stream) {
  static_assert(sizeof(UmmaShared<kStorage, DP>) + 1024 <= 232448, "shared memory of a block");
  constexpr int kBytes = static_cast<int>(sizeof(UmmaShared<kStorage, DP>) + 1024);
  // more than 48 KB is opted into once per device
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> done[kMaxDevices];
  int device = 0;
  cudaError_t error = cudaGetDevice(&device);
  if (error != cudaSuccess) return error;
  if (device < 0 || device >= kMaxDevices || !done[device].load(std::memory_order_acquire)) {
    error = cudaFuncSetAttribute(pool_attn_umma_kernel<kStorage, DP, kTree>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (error != cudaSuccess) return error;
    if (device >= 0 && device < kMaxDevices) done[device].store(true, std::memory_order_release);
  }
  pool_attn_umma_kernel<kStorage, DP, kTree><<<plan.blocks, kUmmaThreads, kBytes, stream>>>(a, plan, status);
  return cudaGetLastError();
}

// Tiles on tcgen05, for plans of kUmmaRows rows per block; one translation unit per way of holding the pool.
template <int kStorage>
cudaError_t launch_umma(const wm_pool_attn_args& a, const Plan& plan, int* status, cudaStream_t stream);

#define WM_POOL_UMMA_UNIT(kStorage)                                                                                                \
  template <>                                                                                                                      \
  cudaError_t launch_umma<kStorage>(const wm_pool_attn_args& a, const Plan& plan, int* status, cudaStream_t stream) {              \
    if (a.ancestors != nullptr)                                                                                                    \
      return a.head_dim <= 64 ? launch_umma_dim<kStorage, 64, true>(a, plan, status, stream) : launch_umma_dim<kStorage, 128, true>(a, plan, status, stream); \
    return a.head_dim <= 64 ? launch_umma_dim<kStorage, 64, false>(a, plan, status, stream) : launch_umma_dim<kStorage, 128, false>(a, plan, status, stream); \
  }

}  // namespace pool
}  // namespace wm
