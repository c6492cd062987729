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
  int group;           // query heads per KV head
  int row_blocks;      // of rows_per_block rows, per KV head
  int rows_per_block;
  int draft_tiles;
  int blocks;   // of the launch: shares, or blocks of all clusters
  int cluster;  // blocks per cluster, 0 where the launch works in shares
  int segment_cost;  // what a segment costs beside its tiles (set-up, joining its warps), in tiles
};

// Slots that the queries of sequence b may see: the dummy and the committed tokens.
__device__ __forceinline__ int visible_slots(const wm_pool_attn_args& a, int b) {
  if (a.lengths == nullptr) return a.k_len;
  return clampi(load_index(a.lengths, a.lengths_is64, b), 0, a.k_len - a.lead) + a.lead;
}

__device__ __forceinline__ int sequence_tiles(const wm_pool_attn_args& a, const Plan& p, int b) {
  const int tiles = (visible_slots(a, b) + kTileKeys - 1) / kTileKeys + p.draft_tiles;
  return max(tiles, 1);  // a segment that sees nothing still writes its zeros
}

// One share: units [begin, end) of `total` (less than 2^31, the host sees to it), and where its first unit lies.
struct Share {
  int total, begin, end;
  int b;        // sequence of unit `begin`
  int b_begin;  // first unit of that sequence
};

// The first unit of a share: equal shares, the first total % shares of them one unit longer.
__device__ __forceinline__ int share_begin(int total, int share, int shares) {
  const int each = total / shares;
  return share * each + min(share, total - each * shares);
}

// The share of block `share`.  Every warp finds it for itself, 32 sequences at a time, so the block does not meet.
__device__ __forceinline__ Share find_share(const wm_pool_attn_args& a, const Plan& p, int share, int shares) {
  const int lane = threadIdx.x & 31, per_tile = a.kv_heads * p.row_blocks;
  Share s;
  int sum = 0;
  for (int b = lane; b < a.batch; b += 32) sum += p.segment_cost + sequence_tiles(a, p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  s.total = sum * per_tile;
  s.begin = share_begin(s.total, share, shares);
  s.end = share_begin(s.total, share + 1, shares);
  s.b = s.b_begin = 0;
  if (s.begin >= s.end) return s;
  for (int base = 0, before = 0; base < a.batch; base += 32) {
    int upto = base + lane < a.batch ? p.segment_cost + sequence_tiles(a, p, base + lane) : 0;
    const int mine = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    upto += before;
    const uint32_t hit = __ballot_sync(0xffffffffu, upto * per_tile > s.begin);
    if (hit != 0) {
      const int at = __ffs(hit) - 1;
      s.b = base + at;
      s.b_begin = __shfl_sync(0xffffffffu, (upto - mine) * per_tile, at);
      break;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return s;
}

// A piece of a segment: tiles [tile, stop) of the `tiles` that segment (b, kv_head, row_block) has.
struct Piece {
  int b, kv_head, row_block;
  int slots;  // visible slots of the sequence
  int past_tiles, tiles;
  int tile, stop;  // empty where the share holds no more than the segment's own cost
  int end;         // first unit behind the piece
};

__device__ __forceinline__ bool whole(const Piece& c) { return c.tile == 0 && c.stop == c.tiles; }

// The piece that starts at unit `at` (at < end) and ends with its segment or with the share; moves (b, b_begin) on.
__device__ __forceinline__ Piece next_piece(const wm_pool_attn_args& a, const Plan& p, int at, int end, int& b, int& b_begin) {
  Piece c;
  const int segments = a.kv_heads * p.row_blocks;
  for (;;) {
    c.slots = visible_slots(a, b);
    c.past_tiles = (c.slots + kTileKeys - 1) / kTileKeys;
    c.tiles = max(c.past_tiles + p.draft_tiles, 1);
    const int b_end = b_begin + (c.tiles + p.segment_cost) * segments;
    if (at < b_end) break;
    b_begin = b_end;
    ++b;
  }
  const int units = c.tiles + p.segment_cost, in = at - b_begin, segment = in / units, first = in - segment * units;
  c.b = b;
  c.kv_head = segment / p.row_blocks;
  c.row_block = segment - c.kv_head * p.row_blocks;
  c.end = min(end, at + units - first);
  c.tile = max(first - p.segment_cost, 0);
  c.stop = max(first + c.end - at - p.segment_cost, 0);
  return c;
}

// Workspace: a note per share, then the partial records, two per share (0: the rest of a segment begun by an earlier
// share, 1: the start of one that a later share ends), each rows_per_block x (reference, sum, head_dim accumulators).
// The note says which segment the share begins and leaves unfinished, and which share ends it (-1: there is none).
struct Note {
  int b, kv_head, row_block, last;
};

__device__ __forceinline__ Note* note_of(const wm_pool_attn_args& a, int share) { return static_cast<Note*>(a.workspace) + share; }

__device__ __forceinline__ float* partial_row(const wm_pool_attn_args& a, const Plan& p, int shares, int share, int which, int row) {
  return reinterpret_cast<float*>(note_of(a, shares)) + ((static_cast<long long>(share) * 2 + which) * p.rows_per_block + row) * (a.head_dim + 2);
}

// One thread of the block notes what its last piece leaves.
__device__ __forceinline__ void leave_note(const wm_pool_attn_args& a, const Share& s, const Piece& c, int share, int shares) {
  Note n = {c.b, c.kv_head, c.row_block, -1};
  if (c.tile == 0 && c.stop < c.tiles) {  // the share that holds the segment's last unit
    const int unit = s.end + c.tiles - c.stop - 1, each = s.total / shares, longer = s.total - each * shares;
    n.last = unit < longer * (each + 1) ? unit / (each + 1) : longer + (unit - longer * (each + 1)) / each;
  }
  *note_of(a, share) = n;
}

__device__ __forceinline__ void row_place(const wm_pool_attn_args& a, const Plan& p, int kv_head, int row_block, int row, int& token, int& head) {
  const int r = row_block * p.rows_per_block + row;
  token = r / p.group;
  head = kv_head * p.group + (r - token * p.group);
}

}  // namespace pool
}  // namespace wm
