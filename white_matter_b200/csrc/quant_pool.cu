// Commit of rows to a pool held in 8 bits, the way back, and the tables of trees of drafted tokens.
#include <limits.h>

#include "serving.cuh"

namespace wm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxGridY = 65535;
constexpr int kMaxPlanes = INT_MAX - kMaxGridY;  // sequences of a commit, (sequence, head) planes of a read back: counted in 32 bits, a grid at a time

// ---------------------------------------------------------------- commit
// 16 bytes of a source row: its values in fp32, and the bits of the largest magnitude as fp32 bits (as integers these order
// like the magnitudes, with infinity and NaN above every number).
template <typename T>
struct Part;
template <>
struct Part<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4& raw, float (&x)[4]) {
    x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y), x[2] = __uint_as_float(raw.z), x[3] = __uint_as_float(raw.w);
  }
  __device__ static uint32_t top(const uint4& raw) {
    return max(max(raw.x & 0x7fffffffu, raw.y & 0x7fffffffu), max(raw.z & 0x7fffffffu, raw.w & 0x7fffffffu));
  }
};
template <>
struct Part<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& raw, float (&x)[8]) {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint32_t top(const uint4& raw) {  // two 16-bit maxima at a time
    const uint32_t m = __vimax3_u16x2(raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu, __vimax3_u16x2(raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu, 0u));
    return max(m << 16, m & 0xffff0000u);
  }
};

// four codes in a word, element 0 in the low byte
template <int kStorage>
__device__ __forceinline__ uint32_t codes_of(const float* x, float inverse) {
  if (kStorage == WM_INT8) {
    // adding 1.5 * 2^23 rounds to an integer, halves to even, and leaves it in the low bits (|x * inverse| < 128); the product
    // is rounded by itself first
    uint32_t n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inverse), 12582912.f));
    return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
  }
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[1] * inverse), "f"(x[0] * inverse));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[3] * inverse), "f"(x[2] * inverse));
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}

// What a row is multiplied by before it is rounded, and the scale that is kept, from the bits of its largest magnitude.
template <int kStorage>
__device__ __forceinline__ void row_scale(uint32_t top, float& inverse, float& scale) {
  inverse = 0.f;
  scale = 0.f;
  if (top >= 0x7f800000u) {
    scale = __uint_as_float(0x7fffffffu);
  } else if (top >= (27u << 23)) {  // 2^-100; below it the quotients would leave the normal range
    if (kStorage == WM_INT8) {  // the correctly rounded quotients are part of the format
      inverse = __fdiv_rn(127.f, __uint_as_float(top));
      scale = __fdiv_rn(__uint_as_float(top), 127.f);
    } else {  // 448 = 1.75 * 2^8
      const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u);
      scale = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      inverse = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    }
  }
}

// LPR lanes hold one row, 16 source bytes each; a thread has its part of kRows rows in flight.  Sources that keep a token's
// heads side by side (kTokens) are read that way, kRows tokens of neighbouring heads; the others slot by slot.  Bound by the
// instructions of a row more than by its bytes (3.3 of 4 per cycle and SM, ALU pipe 65 %, DRAM 52 % of its peak): maxima are taken
// two elements at a time, addresses of a thread's rows in steps of one stride.  A prompt of 8 x 2048 tokens, 128 heads of 64, bf16 to e4m3 (822 MB): 166 us, 4 950
// GB/s (215 us before those two); to int8, whose scale takes two correctly rounded divisions, 196 us.
// grid: (rows of a sequence, sequences, K or V).
constexpr int kRows = 4;

template <typename T, int LPR, int kStorage, bool kTokens>
__global__ void __launch_bounds__(kThreads) pool_commit_kernel(const wm_pool_commit_args a) {
  constexpr int N = Part<T>::N, kGroups = kThreads / LPR;
  constexpr bool kCopy = kStorage == WM_F32 || kStorage == WM_BF16;
  constexpr int kHeld = kCopy ? static_cast<int>(sizeof(T)) : 1;
  const bool values = blockIdx.z != 0;
  const int64_t* pool_strides = values ? a.value_strides : a.key_strides;
  const int64_t* src_strides = values ? a.new_value_strides : a.new_key_strides;
  const int64_t* scale_strides = values ? a.value_scale_strides : a.key_scale_strides;
  const int lane = threadIdx.x % LPR;
  const bool live = lane * N < a.head_dim;
  // the thread's rows: (head, row), (head, row + 1) .. with kTokens, else numbers kGroups apart, head by head
  int head[kRows], row[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (kTokens) {
      const int at = blockIdx.x * kGroups + threadIdx.x / LPR, block = at / a.heads;
      head[i] = at - block * a.heads;
      row[i] = block * kRows + i;
    } else {
      const int at = (blockIdx.x * kRows + i) * kGroups + threadIdx.x / LPR;
      head[i] = at / a.rows;
      row[i] = at - head[i] * a.rows;
    }
  }
  for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const long long first = load_index(a.lengths, a.lengths_is64, b) + a.lead;
    const int count = a.counts != nullptr ? min(a.counts[b], a.rows) : a.rows;
    const T* src = static_cast<const T*>(values ? a.new_values : a.new_keys) + b * src_strides[0] + head[0] * src_strides[1] + lane * N;
    char* pool = static_cast<char*>(values ? a.values : a.keys) + (b * pool_strides[0] + head[0] * pool_strides[1] + (first + row[0]) * pool_strides[2] + lane * N) * kHeld;
    uint4 raw[kRows];
    bool keep[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const long long slot = first + row[i];
      keep[i] = head[i] < a.heads && row[i] < count && slot >= 0 && slot < a.slots;
      int from = row[i];
      if (a.index != nullptr && keep[i]) {
        from = a.index[static_cast<long long>(b) * a.rows + row[i]];
        keep[i] = from >= 0 && from < a.source_rows;
      }
      raw[i] = make_uint4(0, 0, 0, 0);
      if (keep[i] && live) raw[i] = *reinterpret_cast<const uint4*>(src + (kTokens ? 0 : (head[i] - head[0]) * src_strides[1]) + from * src_strides[2]);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      char* dst = pool + (kTokens ? i * pool_strides[2] : (head[i] - head[0]) * pool_strides[1] + (row[i] - row[0]) * pool_strides[2]) * kHeld;
      if (kCopy) {
        if (keep[i] && live) *reinterpret_cast<uint4*>(dst) = raw[i];
        continue;
      }
      uint32_t top = Part<T>::top(raw[i]);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      float inverse, scale;
      row_scale<kStorage>(top, inverse, scale);
      if (!keep[i]) continue;
      if (live) {
        float x[N];
        Part<T>::unpack(raw[i], x);
        uint32_t w[N / 4];
#pragma unroll
        for (int e = 0; e < N / 4; ++e) w[e] = codes_of<kStorage>(x + 4 * e, inverse);
        if (inverse == 0.f) {  // a row of zeros, or one that is not finite
#pragma unroll
          for (int e = 0; e < N / 4; ++e) w[e] = 0;
        }
        if (N == 8)
          *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[N / 4 - 1]);
        else
          *reinterpret_cast<uint32_t*>(dst) = w[0];
      }
      if (lane == 0) {
        float* scales = values ? a.value_scales : a.key_scales;
        scales[b * scale_strides[0] + head[i] * scale_strides[1] + (first + row[i]) * scale_strides[2]] = scale;
      }
    }
  }
}

template <typename T, int LPR, int kStorage>
int commit_storage(const wm_pool_commit_args& a, cudaStream_t stream) {
  const bool tokens = a.rows >= kRows && a.new_key_strides[1] < a.new_key_strides[2];
  const long long rows = static_cast<long long>(a.heads) * (tokens ? (a.rows + kRows - 1) / kRows * kRows : a.rows);
  const long long per_block = kRows * kThreads / LPR;
  const dim3 grid(static_cast<unsigned>((rows + per_block - 1) / per_block), static_cast<unsigned>(a.batch < kMaxGridY ? a.batch : kMaxGridY), 2);
  if (tokens)
    pool_commit_kernel<T, LPR, kStorage, true><<<grid, kThreads, 0, stream>>>(a);
  else
    pool_commit_kernel<T, LPR, kStorage, false><<<grid, kThreads, 0, stream>>>(a);
  count_launch();
  return cuda_check(cudaGetLastError(), "pool_commit_kernel");
}

template <typename T, int LPR>
int commit(const wm_pool_commit_args& a, cudaStream_t stream) {
  if (a.storage == WM_INT8) return commit_storage<T, LPR, WM_INT8>(a, stream);
  if (a.storage == WM_E4M3) return commit_storage<T, LPR, WM_E4M3>(a, stream);
  return commit_storage<T, LPR, sizeof(T) == 4 ? WM_F32 : WM_BF16>(a, stream);
}

int commit_rows(const wm_pool_commit_args& a, cudaStream_t stream) {
  const int lanes = a.head_dim * (a.dtype == WM_F32 ? 4 : 2) / 16;
  if (a.dtype == WM_F32) return lanes <= 8 ? commit<float, 8>(a, stream) : lanes <= 16 ? commit<float, 16>(a, stream) : commit<float, 32>(a, stream);
  return lanes <= 8 ? commit<__nv_bfloat16, 8>(a, stream) : commit<__nv_bfloat16, 16>(a, stream);
}

// The lengths behind a commit, a warp per sequence: a launch and dependent loads, 1.5 us for 64 sequences with 33 picked rows.
__global__ void __launch_bounds__(kThreads) pool_advance_kernel(void* lengths, int lengths_is64, const int32_t* index, const int32_t* counts, int batch, int rows,
                                                                int source_rows, int capacity) {
  const int lane = threadIdx.x & 31;
  const long long b = static_cast<long long>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (b >= batch) return;
  int written = counts != nullptr ? min(max(counts[b], 0), rows) : rows;
  if (index != nullptr) {
    for (int base = 0; base < written; base += 32) {
      const int i = base + lane, from = i < written ? index[b * rows + i] : 0;
      const uint32_t outside = __ballot_sync(0xffffffffu, from < 0 || from >= source_rows);
      if (outside != 0) written = min(written, base + __ffs(outside) - 1);
    }
  }
  if (lane != 0) return;
  const long long before = load_index(lengths, lengths_is64, static_cast<int>(b)), after = min(before + written, static_cast<long long>(capacity));
  if (lengths_is64)
    static_cast<long long*>(lengths)[b] = after;
  else
    static_cast<int*>(lengths)[b] = static_cast<int>(after);
}

// ---------------------------------------------------------------- read back
// Bound by HBM, two thirds of it writes.  A plane is one (b, head).  A thread turns 16 codes of kUnits rows, all in flight
// together; the threads of a block that do not fill a row are idle.  A pool of 16 x 128 heads x 2049 rows of 64, e4m3 to bf16
// (1.36 GB): 240 us, 5 650 GB/s; eight codes and four rows per thread, whose loads are narrower: 312 us.
constexpr int kUnits = 2;

template <typename T>
__global__ void __launch_bounds__(kThreads) pool_dequant_kernel(const wm_pool_dequant_args a) {
  const int per_row = a.head_dim / 16, rows = kThreads / per_row, row = threadIdx.x / per_row, piece = threadIdx.x - row * per_row;
  if (row >= rows) return;
  for (int plane = blockIdx.y; plane < a.batch * a.heads; plane += gridDim.y) {
    const int b = plane / a.heads, h = plane - b * a.heads;
    const long long end = a.lengths == nullptr ? a.slots : load_index(a.lengths, a.lengths_is64, b) + a.lead;
    const char* codes = static_cast<const char*>(a.codes) + b * a.code_strides[0] + h * a.code_strides[1] + 16 * piece;
    const float* scales = a.scales + b * a.scale_strides[0] + h * a.scale_strides[1];
    T* out = static_cast<T*>(a.out) + b * a.out_strides[0] + h * a.out_strides[1] + 16 * piece;
    uint4 raw[kUnits];
    float scale[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int slot = (blockIdx.x * kUnits + i) * rows + row;
      raw[i] = make_uint4(0, 0, 0, 0);
      scale[i] = 0.f;
      if (slot < a.slots && slot < end) {
        raw[i] = *reinterpret_cast<const uint4*>(codes + slot * a.code_strides[2]);
        scale[i] = scales[slot * a.scale_strides[2]];
      }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int slot = (blockIdx.x * kUnits + i) * rows + row;
      if (slot >= a.slots) continue;
      const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
      constexpr int N = 32 / sizeof(T);  // one 32-byte store
#pragma unroll
      for (int q = 0; q < 16 / N; ++q) {
        __align__(16) T y[N];
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          float x[4];
          codes_to_float(w[(q * N + j) / 4], a.storage == WM_INT8, x);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[j + e] = from_float<T>(x[e] * scale[i]);
        }
        uint4* dst = reinterpret_cast<uint4*>(out + slot * a.out_strides[2] + q * N);
        __stcs(dst, reinterpret_cast<const uint4*>(y)[0]);
        __stcs(dst + 1, reinterpret_cast<const uint4*>(y)[1]);
      }
    }
  }
}

// ---------------------------------------------------------------- tree tables
// Latency: a launch and log2(depth) rounds of shared memory; 3.5 us for one tree of 8 nodes, 6.5 us for 128 of 256.
// Pointer doubling over bit sets: after r rounds a node knows its 2^r nearest ancestors and the one 2^r steps up, and
// takes over that one's set in the next round.  One block per tree, one thread per node; a round reads its neighbours'
// state, meets, and writes.  Chains that have not ended after the rounds a chain of `tokens` nodes takes are cycles.
constexpr int kTreeWords = kMaxTreeNodes / 32;
constexpr int kRoot = -1, kDead = -2;

__global__ void draft_tree_kernel(const wm_draft_tree_args a, int rounds) {
  __shared__ uint32_t sets[kTreeWords][kMaxTreeNodes];
  __shared__ int jumps[kMaxTreeNodes];
  const int node = threadIdx.x, words = (a.tokens + 31) / 32;
  const long long row = static_cast<long long>(blockIdx.x) * a.tokens + node;
  const bool live = node < a.tokens;
  int jump = kDead;
  uint32_t set[kTreeWords];
#pragma unroll
  for (int w = 0; w < kTreeWords; ++w) set[w] = 0;
  if (live) {
    const int parent = a.parents[row];
    jump = parent == -1 ? kRoot : (parent >= 0 && parent < a.tokens && parent != node ? parent : kDead);
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) {
      if (jump >= 0 && (jump >> 5) == w) set[w] = 1u << (jump & 31);
      if (w < words) sets[w][node] = set[w];
    }
    jumps[node] = jump;
  }
  for (int r = 0; r < rounds; ++r) {
    if (!__syncthreads_or(jump >= 0)) break;  // also: every node's state of the last round is in place
    const int via = jump;
    if (via >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w)
        if (w < words) set[w] |= sets[w][via];
      jump = jumps[via];
    }
    __syncthreads();
    if (via >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w)
        if (w < words) sets[w][node] = set[w];
      jumps[node] = jump;
    }
  }
  if (!live) return;
  int depth = 0;
#pragma unroll
  for (int w = 0; w < kTreeWords; ++w) {
    if (w < words) {
      depth += __popc(set[w]);
      uint32_t seen = jump == kRoot ? set[w] : 0u;
      if (a.include_self && jump == kRoot && (node >> 5) == w) seen |= 1u << (node & 31);
      a.ancestors[row * words + w] = seen;
    }
  }
  a.depths[row] = jump == kRoot ? depth : -1;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned16(const int64_t* strides, int esize) {
  return strides[0] * esize % 16 == 0 && strides[1] * esize % 16 == 0 && strides[2] * esize % 16 == 0;
}

}  // namespace

int pool_commit_launch(const wm_pool_commit_args& a, cudaStream_t stream) {
  const char* who = "wm_pool_commit";
  if (a.keys == nullptr || a.values == nullptr || a.new_keys == nullptr || a.new_values == nullptr || a.lengths == nullptr)
    return fail(WM_EINVAL, "%s: pool, new rows and lengths are required", who);
  if (a.dtype != WM_F32 && a.dtype != WM_BF16) return fail(WM_EINVAL, "%s: new rows must be WM_F32 or WM_BF16", who);
  const bool quantised = a.storage == WM_INT8 || a.storage == WM_E4M3;
  if (!quantised && a.storage != a.dtype) return fail(WM_EINVAL, "%s: the pool must be WM_INT8, WM_E4M3 or of the rows' type", who);
  if (quantised && (a.key_scales == nullptr || a.value_scales == nullptr)) return fail(WM_EINVAL, "%s: an 8-bit pool needs its scales", who);
  if (a.batch < 1 || a.heads < 1 || a.slots < 1 || a.rows < 1 || a.source_rows < 1 || a.head_dim < 1)
    return fail(WM_EINVAL, "%s: sizes must be positive", who);
  if (a.index == nullptr && a.source_rows < a.rows) return fail(WM_EINVAL, "%s: more rows than the source has", who);
  if (a.lead != 0 && a.lead != 1) return fail(WM_EINVAL, "%s: lead must be 0 or 1", who);
  if (a.head_dim % 16 || a.head_dim > 128) return fail(WM_EUNSUPPORTED, "%s: head_dim must be a multiple of 16 up to 128", who);
  if (a.batch > kMaxPlanes) return fail(WM_EUNSUPPORTED, "%s: too many sequences", who);
  if (static_cast<long long>(a.heads) * a.rows > INT_MAX - kRows * kThreads) return fail(WM_EUNSUPPORTED, "%s: too many rows per sequence", who);
  const int wide = a.dtype == WM_F32 ? 4 : 2, held = quantised ? 1 : wide;
  if (!aligned16(a.keys) || !aligned16(a.values) || !aligned16(a.new_keys) || !aligned16(a.new_values) || !aligned16(a.key_strides, held) ||
      !aligned16(a.value_strides, held) || !aligned16(a.new_key_strides, wide) || !aligned16(a.new_value_strides, wide))
    return fail(WM_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
  return commit_rows(a, stream);
}

int pool_advance_launch(void* lengths, int lengths_is64, const int32_t* index, const int32_t* counts, int batch, int rows, int source_rows, int capacity, cudaStream_t stream) {
  const char* who = "wm_pool_advance";
  if (lengths == nullptr) return fail(WM_EINVAL, "%s: lengths are required", who);
  if (batch < 1 || rows < 1 || source_rows < 1 || capacity < 1) return fail(WM_EINVAL, "%s: sizes must be positive", who);
  if (rows > INT_MAX - 32) return fail(WM_EUNSUPPORTED, "%s: too many rows per sequence", who);
  pool_advance_kernel<<<static_cast<unsigned>((static_cast<long long>(batch) + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, stream>>>(
      lengths, lengths_is64, index, counts, batch, rows, source_rows, capacity);
  count_launch();
  return cuda_check(cudaGetLastError(), "pool_advance_kernel");
}

int pool_dequant_launch(const wm_pool_dequant_args& a, cudaStream_t stream) {
  const char* who = "wm_pool_dequant";
  if (a.codes == nullptr || a.scales == nullptr || a.out == nullptr) return fail(WM_EINVAL, "%s: codes, scales and out are required", who);
  if (a.storage != WM_INT8 && a.storage != WM_E4M3) return fail(WM_EINVAL, "%s: storage must be WM_INT8 or WM_E4M3", who);
  if (a.dtype != WM_F32 && a.dtype != WM_BF16) return fail(WM_EINVAL, "%s: dtype must be WM_F32 or WM_BF16", who);
  if (a.batch < 1 || a.heads < 1 || a.slots < 1 || a.head_dim < 1) return fail(WM_EINVAL, "%s: sizes must be positive", who);
  if (a.lead != 0 && a.lead != 1) return fail(WM_EINVAL, "%s: lead must be 0 or 1", who);
  if (a.head_dim % 16 || a.head_dim > 128) return fail(WM_EUNSUPPORTED, "%s: head_dim must be a multiple of 16 up to 128", who);
  const long long planes = static_cast<long long>(a.batch) * a.heads;
  if (planes > kMaxPlanes) return fail(WM_EUNSUPPORTED, "%s: too many (sequence, head) planes", who);
  if (a.slots > kMaxSlots) return fail(WM_EUNSUPPORTED, "%s: too many slots", who);
  const int wide = a.dtype == WM_F32 ? 4 : 2;
  if (!aligned16(a.codes) || !aligned16(a.out) || !aligned16(a.code_strides, 1) || !aligned16(a.out_strides, wide))
    return fail(WM_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
  const int per_block = kUnits * (kThreads / (a.head_dim / 16));
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.slots) + per_block - 1) / per_block), static_cast<unsigned>(planes < kMaxGridY ? planes : kMaxGridY));
  if (a.dtype == WM_F32)
    pool_dequant_kernel<float><<<grid, kThreads, 0, stream>>>(a);
  else
    pool_dequant_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(a);
  count_launch();
  return cuda_check(cudaGetLastError(), "pool_dequant_kernel");
}

int draft_tree_launch(const wm_draft_tree_args& a, cudaStream_t stream) {
  const char* who = "wm_draft_tree";
  if (a.parents == nullptr || a.ancestors == nullptr || a.depths == nullptr) return fail(WM_EINVAL, "%s: parents, ancestors and depths are required", who);
  if (a.batch < 1 || a.tokens < 1) return fail(WM_EINVAL, "%s: sizes must be positive", who);
  if (a.tokens > kMaxTreeNodes) return fail(WM_EUNSUPPORTED, "%s: at most %d drafted tokens", who, kMaxTreeNodes);
  if (a.include_self != 0 && a.include_self != 1) return fail(WM_EINVAL, "%s: include_self must be 0 or 1", who);
  int rounds = 0;
  while ((1 << rounds) < a.tokens) ++rounds;
  draft_tree_kernel<<<a.batch, (a.tokens + 31) / 32 * 32, 0, stream>>>(a, rounds);
  count_launch();
  return cuda_check(cudaGetLastError(), "draft_tree_kernel");
}

}  // namespace wm

extern "C" {

int wm_pool_commit(const wm_pool_commit_args* a, void* stream) {
  if (a == nullptr) return wm::fail(WM_EINVAL, "wm_pool_commit: null arguments");
  return wm::pool_commit_launch(*a, static_cast<cudaStream_t>(stream));
}

int wm_pool_advance(void* lengths, int32_t lengths_is64, const int32_t* index, const int32_t* counts, int32_t batch, int32_t rows, int32_t source_rows,
                    int32_t capacity, void* stream) {
  return wm::pool_advance_launch(lengths, lengths_is64, index, counts, batch, rows, source_rows, capacity, static_cast<cudaStream_t>(stream));
}

int wm_pool_dequant(const wm_pool_dequant_args* a, void* stream) {
  if (a == nullptr) return wm::fail(WM_EINVAL, "wm_pool_dequant: null arguments");
  return wm::pool_dequant_launch(*a, static_cast<cudaStream_t>(stream));
}

int wm_draft_tree(const wm_draft_tree_args* a, void* stream) {
  if (a == nullptr) return wm::fail(WM_EINVAL, "wm_draft_tree: null arguments");
  return wm::draft_tree_launch(*a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
