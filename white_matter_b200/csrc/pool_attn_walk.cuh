// How the blocks of the pool attention share the work, common to its kernels.
//
// The rows of one KV head are its queries, (token, head of the group) with the head running faster, cut into row
// blocks.  A segment is one (sequence, KV head, row block); it walks the sequence's visible slots and then the drafted
// tokens in tiles of kTileKeys.  The tiles of all segments, laid end to end, are cut into equal shares, one per block
// of a single wave, whatever the lengths are: they are read on the device, so the launch can be captured and replayed
// while they grow.  A segment inside one share is written out by its block.  One that crosses shares leaves a partial
// record (reference, sum and accumulator of every row) per share, and a second kernel joins the records of a segment.
#pragma once

#include "serving.cuh"

namespace wm {
namespace pool {

constexpr int kTileKeys = 128;
constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;

struct Plan {
  int row_blocks;      // of rows_per_block rows, per KV head
  int rows_per_block;
  int draft_tiles;
};

// Slots that the queries of sequence b may see: the dummy and the committed tokens.
__device__ __forceinline__ int visible_slots(const wm_pool_attn_args& a, int b) {
  if (a.lengths == nullptr) return a.k_len;
  return clampi(load_index(a.lengths, a.lengths_is64, b), 0, a.k_len - a.lead) + a.lead;
}

__device__ __forceinline__ int sequence_tiles(const wm_pool_attn_args& a, const Plan& p, int b) {
  const int tiles = (visible_slots(a, b) + kTileKeys - 1) / kTileKeys + p.draft_tiles;
  return tiles > 0 ? tiles : 1;  // a segment that sees nothing still writes its zeros
}

// One share: units [begin, end) of `total`, and where its first unit lies.
struct Share {
  long long total, begin, end;
  int b;               // sequence of unit `begin`
  long long b_begin;   // first unit of that sequence
};

__device__ __forceinline__ long long share_begin(long long total, int share, int shares) { return total * share / shares; }

// Inclusive prefix sum over the block, and the block's total; `sums` holds kWarps values.
__device__ __forceinline__ long long block_scan(long long x, long long* sums, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) x += sums[w];
    total += sums[w];
  }
  return x;
}

// The share of block `share`; all threads of the block call it.
__device__ __forceinline__ Share find_share(const wm_pool_attn_args& a, const Plan& p, int share, int shares) {
  __shared__ long long sums[kWarps];
  __shared__ long long found_begin;
  __shared__ int found;
  const long long per_tile = static_cast<long long>(a.kv_heads) * p.row_blocks;
  Share s;
  s.total = 0;
  for (int base = 0; base < a.batch; base += kThreads) {
    const int b = base + threadIdx.x;
    long long chunk;
    block_scan(b < a.batch ? sequence_tiles(a, p, b) : 0, sums, chunk);
    s.total += chunk * per_tile;
  }
  s.begin = share_begin(s.total, share, shares);
  s.end = share_begin(s.total, share + 1, shares);
  long long before = 0;
  for (int base = 0; base < a.batch; base += kThreads) {
    const int b = base + threadIdx.x;
    const long long mine = b < a.batch ? sequence_tiles(a, p, b) : 0;
    long long chunk;
    const long long upto = (before + block_scan(mine, sums, chunk)) * per_tile;
    if (s.begin < upto && s.begin >= upto - mine * per_tile) {
      found = b;
      found_begin = upto - mine * per_tile;
    }
    before += chunk;
  }
  __syncthreads();
  s.b = found;
  s.b_begin = found_begin;
  return s;
}

// A piece of a segment: tiles [tile, stop) of the `tiles` that segment (b, kv_head, row_block) has.
struct Piece {
  int b, kv_head, row_block;
  int slots;  // visible slots of the sequence
  int past_tiles, tiles;
  int tile, stop;
};

__device__ __forceinline__ bool whole(const Piece& c) { return c.tile == 0 && c.stop == c.tiles; }

// The piece that starts at unit `at` (at < s.end) and ends with its segment or with the share; moves (b, b_begin) on.
__device__ __forceinline__ Piece next_piece(const wm_pool_attn_args& a, const Plan& p, long long at, long long end, int& b, long long& b_begin) {
  Piece c;
  const int segments = a.kv_heads * p.row_blocks;
  for (;;) {
    c.slots = visible_slots(a, b);
    c.past_tiles = (c.slots + kTileKeys - 1) / kTileKeys;
    c.tiles = c.past_tiles + p.draft_tiles;
    if (c.tiles < 1) c.tiles = 1;
    const long long b_end = b_begin + static_cast<long long>(c.tiles) * segments;
    if (at < b_end) break;
    b_begin = b_end;
    ++b;
  }
  const long long in = at - b_begin;
  const int segment = static_cast<int>(in / c.tiles);
  c.b = b;
  c.tile = static_cast<int>(in - static_cast<long long>(segment) * c.tiles);
  c.kv_head = segment / p.row_blocks;
  c.row_block = segment - c.kv_head * p.row_blocks;
  const long long room = end - at;
  c.stop = room < c.tiles - c.tile ? c.tile + static_cast<int>(room) : c.tiles;
  return c;
}

// Partial records: two per share (0: the rest of a segment begun by an earlier share, 1: the start of one that a
// later share ends), each rows_per_block x (reference, sum, head_dim accumulators).
__device__ __forceinline__ float* partial_row(float* workspace, const wm_pool_attn_args& a, const Plan& p, int share, int which, int row) {
  return workspace + ((static_cast<long long>(share) * 2 + which) * p.rows_per_block + row) * (a.head_dim + 2);
}

__device__ __forceinline__ void row_place(const wm_pool_attn_args& a, const Piece& c, const Plan& p, int row, int& token, int& head) {
  const int group = a.q_heads / a.kv_heads, r = c.row_block * p.rows_per_block + row;
  token = r / group;
  head = c.kv_head * group + (r - token * group);
}

}  // namespace pool
}  // namespace wm
