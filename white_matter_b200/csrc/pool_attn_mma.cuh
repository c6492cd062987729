// Pool attention for bf16 queries with up to 16 rows per KV head, on the warp-level matrix instructions (bf16 operands, fp32 sums).
//
// The read is bound by HBM: a pool row is used by the few rows of its KV head and then never again, so what counts is
// bytes in flight, and few instructions per byte.  Pool rows therefore go from global memory straight into the registers
// of the warp that uses them, in the order the matrix instruction wants them, and the next step's rows are asked for as
// soon as this step's have been used; shared memory only joins the warps of a block at the end of a segment.
//
// Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that the keys (or head_dim) fill the 16 rows
// of an instruction and 8 query rows its columns: a single query wastes 7 of 8 columns instead of 15 of 16, registers
// grow by 8 rows at a time, and the fragment of K that a lane needs is one contiguous piece of a pool row.  The order of
// head_dim inside the instructions is free as long as Q (or the output) follows it: lane t of a row's four lanes holds
// elements t*DP/4 .. of a key, lane g of eight holds elements g*DP/8 .. of a value row.
//
// Codes of 8-bit pools become bf16 in registers, which is exact; the key's scale multiplies the score in fp32, the
// value's scale the weight.  Weights over bf16 pools are rounded to bf16 (2^-8 of themselves at most), and the sum takes them as
// rounded.  Over 8-bit pools they enter the product in two parts, rounded and rest, 16 bits together: with one part, reads of one
// sequence were 1.2 to 1.5 times as far from the exact result as the output's rounding, with two 1.0, for 5 % of the time of
// 64 sequences (115.6 -> 121 us) and none on one.  (Over bf16 pools an infinity's product with the rest would be NaN.)
//
// A row's weights are exponentials against a reference that moves only when a score exceeds it by 8 (in powers of two), so the
// common step needs one vote instead of a reduction over the lanes.  Weights up to 2^8 lose no precision (the sums are fp32), but range:
// values above 2^118 in magnitude may overflow sums whose mean does not, and weights below 2^-118 of a row's largest are lost.
//
// 64 sequences of up to 8192 tokens, 16 heads of 64, one token: 122 us over int8 (4 690 GB/s), 133 us over e4m3.  No unit is full there (2.2
// instructions per cycle and SM of 4, ALU pipe 55 %, tensor pipe 21 %, DRAM 72 % of the copy bandwidth): what is left is latency, of memory before all, that 16
// warps per SM do not cover, and every instruction more shows.  Heads of 128, 4 per KV head: 130 and 141 us for 3 % fewer bytes.  bf16
// with 8 drafted tokens 163 to 174 us (6 600 to 6 190 GB/s), bound by HBM.  One sequence of 480 tokens: 5.6 us.
#pragma once

#include <math.h>

#include "pool_attn_walk.cuh"
#include "sm100_ptx.cuh"

namespace wm {
namespace pool {

constexpr float kNoReference = -3.0e38f;
constexpr float kReferenceSlack = 8.f;

// ---------------------------------------------------------------- instructions
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first product of a sum: nothing to add to
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// within 2^-23 of the quotient: a weight is read back from its 8 bits with it
__device__ __forceinline__ float reciprocal_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
// (a & b) | c as one instruction: written as operators with two constants it becomes two, and the conversion of int8 codes is
// what the 8-bit read spends most of its instructions on (64 sequences of up to 8192 rows: 152 us against 122 us)
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(a), "r"(b), "r"(c));
  return y;
}
// kBytes (4, 8 or 16) of a pool row; read once, so kept out of L1
template <int kBytes>
__device__ __forceinline__ void load_row(uint32_t* r, const char* p) {
  if (kBytes == 16)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[kBytes / 4 > 1]), "=r"(r[kBytes / 4 > 2 ? 2 : 0]), "=r"(r[kBytes / 4 > 3 ? 3 : 0]) : "l"(p));
  else if (kBytes == 8)
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[kBytes / 4 > 1]) : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r[0]) : "l"(p));
}

// ---------------------------------------------------------------- how rows are held
template <int kStorage>
struct Codes {
  static constexpr int kBytes = kStorage == WM_BF16 ? 2 : 1;
  // e4m3's two NaN codes come out of pairs() as +-480, which no other code is: `top`, the largest magnitude that it met, tells whether
  // there were any.  Who finds some sees to what he made of them.  (64 sequences of up to 8192 rows of 64, one token: 123 -> 133 us.  NaN
  // made in place, by zero times a product that overflows for 480 alone, took 142 us, a vote in every step 136 us.)
  __device__ static bool some_nan(uint32_t top) { return kStorage == WM_E4M3 && ((top & 0xffffu) == 0x07f0u || top >> 16 == 0x07f0u); }
  // bit 7 of every byte that is a NaN code
  __device__ static uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
  // a pair with NaN for +-480
  __device__ static uint32_t repaired(uint32_t pair) {
    if ((pair & 0x7fffu) == 0x43f0u) pair |= 0x7fffu;
    if ((pair & 0x7fff0000u) == 0x43f00000u) pair |= 0x7fff0000u;
    return pair;
  }
  // bytes 0, 2 (even) and 1, 3 (odd) of a word of codes as bf16 pairs
  __device__ static void pairs(uint32_t w, uint32_t& even, uint32_t& odd, uint32_t& top) {
    if (kStorage == WM_INT8) {
      even = int8_pair(w);
      odd = int8_pair(w >> 8);
    } else {
      const uint32_t e = w << 4 & 0x07f007f0u, o = w >> 4 & 0x07f007f0u;
      top = __vimax3_u16x2(top, e, o);
      even = e4m3_pair(e, w << 8);
      odd = e4m3_pair(o, w);
    }
  }

 private:
  // low seven bits as 128 + x, the sign bit as -128 or -256: their sum is the code, exactly
  __device__ static uint32_t int8_pair(uint32_t w) {
    const uint32_t x = and_or(w, 0x007f007fu, 0x43004300u), s = and_or(w, 0x00800080u, 0xc300c300u);
    uint32_t y;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(x), "r"(0x3f803f80u), "r"(s));
    return y;
  }
  // exponent and fraction in the places bf16 has them, which reads as 2^-120 of the number (subnormals too)
  __device__ static uint32_t e4m3_pair(uint32_t magnitude, uint32_t sign) {
    const uint32_t x = and_or(sign, 0x80008000u, magnitude);
    uint32_t y;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x7b807b80u));
    return y;
  }
};

// A lane's part of 16 pool rows: two key rows (g, g + 8) in pieces of DP/4 elements, four value rows (2t, 2t + 1, 2t + 8,
// 2t + 9) in pieces of DP/8.
template <int kStorage, int DP>
struct Rows {
  static constexpr int kBytes = Codes<kStorage>::kBytes;
  static constexpr int kKeyBytes = DP / 4 * kBytes, kValueBytes = DP / 8 * kBytes;
  static constexpr int kKeyWords = kKeyBytes / 4, kValueWords = kValueBytes / 4;
  static constexpr int kKeyUnit = kKeyBytes % 16 ? 8 : 16;
  static constexpr int kValueUnit = kValueBytes % 16 == 0 ? 16 : (kValueBytes % 8 == 0 ? 8 : 4);

  // Where the piece of lane t (key rows) or g (value rows) starts.  A row of fewer than DP elements (row_bytes, a multiple of
  // 16) has no whole piece for its last lanes: they read the last piece of the row instead.  What two lanes read then
  // counts once, for the lower one: the queries are zero for it in the other lane, and its sums are not stored.
  __device__ static int key_piece(int t, int row_bytes) { return min(t * kKeyBytes, row_bytes - kKeyBytes); }
  __device__ static int value_piece(int g, int row_bytes) { return min(g * kValueBytes, row_bytes - kValueBytes); }

  __device__ static void load_key(uint32_t (&r)[kKeyWords], const char* piece) {
#pragma unroll
    for (int i = 0; i < kKeyBytes / kKeyUnit; ++i) load_row<kKeyUnit>(r + i * kKeyUnit / 4, piece + i * kKeyUnit);
  }
  __device__ static void load_value(uint32_t (&r)[kValueWords], const char* piece) {
#pragma unroll
    for (int i = 0; i < kValueBytes / kValueUnit; ++i) load_row<kValueUnit>(r + i * kValueUnit / 4, piece + i * kValueUnit);
  }
  // Fragment s (16 of head_dim) of K: elements 4s .. 4s + 3 of the piece.  8-bit pools take them in the order 0, 2, 1, 3,
  // which is how a word of codes comes apart; kPermute gives bf16 rows the same order.
  template <bool kPermute>
  __device__ static void key_fragment(uint32_t (&a)[4], const uint32_t (&lo)[kKeyWords], const uint32_t (&hi)[kKeyWords], int s, uint32_t& top) {
    if (kStorage == WM_BF16) {
      const uint32_t l0 = lo[2 * s < kKeyWords ? 2 * s : 0], l1 = lo[2 * s + 1 < kKeyWords ? 2 * s + 1 : 0];
      const uint32_t h0 = hi[2 * s < kKeyWords ? 2 * s : 0], h1 = hi[2 * s + 1 < kKeyWords ? 2 * s + 1 : 0];
      a[0] = kPermute ? __byte_perm(l0, l1, 0x5410) : l0;
      a[1] = kPermute ? __byte_perm(h0, h1, 0x5410) : h0;
      a[2] = kPermute ? __byte_perm(l0, l1, 0x7632) : l1;
      a[3] = kPermute ? __byte_perm(h0, h1, 0x7632) : h1;
    } else {
      Codes<kStorage>::pairs(lo[s], a[0], a[2], top);
      Codes<kStorage>::pairs(hi[s], a[1], a[3], top);
    }
  }
  // Fragment s of V^T: elements 2s, 2s + 1 of the piece for the four keys.
  __device__ static void value_fragment(uint32_t (&a)[4], const uint32_t (&v)[4][kValueWords], int s, uint32_t& top) {
    if (kStorage == WM_BF16) {
      const int w = s < kValueWords ? s : 0;
      a[0] = __byte_perm(v[0][w], v[1][w], 0x5410);
      a[1] = __byte_perm(v[0][w], v[1][w], 0x7632);
      a[2] = __byte_perm(v[2][w], v[3][w], 0x5410);
      a[3] = __byte_perm(v[2][w], v[3][w], 0x7632);
    } else {
      const uint32_t pick = s & 1 ? 0x7632 : 0x5410;  // elements 2s, 2s + 1 of two keys: x0 x1 y0 y1
      const uint32_t first = __byte_perm(v[0][s / 2], v[1][s / 2], pick), second = __byte_perm(v[2][s / 2], v[3][s / 2], pick);
      Codes<kStorage>::pairs(first, a[0], a[1], top);
      Codes<kStorage>::pairs(second, a[2], a[3], top);
    }
  }
};

// ---------------------------------------------------------------- state of a warp
template <int DP, int RT>
struct State {
  float o[DP / 16][RT][4];  // O^T: head_dim g*DP/8 + 2s (+1), rows 2t, 2t + 1 of tile rt
  float m[RT][2], l[RT][2]; // reference and this lane's part of the sum, rows 2t and 2t + 1
  uint32_t fresh;           // bit 2 rt + j: row 2t + j of tile rt has seen no key yet (its reference is 0)
};

// Queries as B operands of S^T = K Q^T: rows g of tile rt, fragment s.  Few tiles stay in registers, more lie in shared memory.
template <int DP, int RT>
struct Queries {
  static constexpr bool kShared = RT * DP > 128;
  uint2 reg[kShared ? 1 : RT][kShared ? 1 : DP / 16];
  const uint2* shared;
  __device__ uint2 get(int rt, int s) const { return kShared ? shared[(rt * (DP / 16) + s) * 32 + (threadIdx.x & 31)] : reg[kShared ? 0 : rt][kShared ? 0 : s]; }
};

// Products of 16 keys with the queries of every tile: S^T, keys g and g + 8 in the rows of x.
template <int kStorage, int DP, int RT, bool kPermute>
__device__ __forceinline__ void scores(const uint32_t (&kr)[2][Rows<kStorage, DP>::kKeyWords], const Queries<DP, RT>& q, float (&x)[RT][4], uint32_t& top) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    uint32_t ka[4];
    Rows<kStorage, DP>::template key_fragment<kPermute>(ka, kr[0], kr[1], s, top);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const uint2 b = q.get(rt, s);
      if (s == 0)
        mma_16816_first(x[rt], ka[0], ka[1], ka[2], ka[3], b.x, b.y);
      else
        mma_16816(x[rt], ka[0], ka[1], ka[2], ka[3], b.x, b.y);
    }
  }
}

// What 16 keys bring along: factor of the score and scale of the value for keys g and g + 8, and whether every row sees all
// 16 of them (else bit 0 / 1 of `seen` says whether row 2t + j sees key g / g + 8).
struct Keys {
  float factor[2], scale[2];
  bool all;
};

// The value scale of a key: a row that is not seen may have any, which becomes 1.
__device__ __forceinline__ float usable_scale(float scale, bool seen) { return seen ? scale : 1.f; }

// Below this scale a weight that counts in the sum may be lost in its product with the scale (products below 2^-126 are zero): such keys,
// rows of zeros with scale 0 among them, enter the sum by the weight itself.  From it on, only weights below 2^-62 are lost.  (64
// sequences with 32 drafted tokens over int8 rows of 64: 287 -> 294 us for looking; heads of 128: no difference.)
constexpr float kTinyScale = 0x1p-64f;

// Weights of U x 16 keys for every tile, as B operands of O^T += V^T P^T.  x holds the keys' products with the queries (keys
// g: x[.][.][0], [1]; g + 8: [2], [3]; rows 2t, 2t + 1).  With kFine the weights come in two parts, rounded (pb) and what the
// rounding left (rest).
template <int DP, int RT, int U, bool kScaled, bool kPerRow, bool kFine = false>
__device__ __forceinline__ void weights(State<DP, RT>& st, float (&x)[U][RT][4], const Keys (&keys)[U], const uint32_t (&seen)[U][kPerRow ? RT : 1][2], uint32_t (&pb)[U][RT][2],
                                        uint32_t (*rest)[RT][2] = nullptr) {
  // x becomes the exponent against the row's reference; -infinity where the row does not see the key
  float over = -INFINITY;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float(&y)[4] = x[u][rt];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = fmaf(y[e], keys[u].factor[e >> 1], -st.m[rt][e & 1]);
      if (!keys[u].all) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!(seen[u][kPerRow ? rt : 0][e & 1] >> (e >> 1) & 1u)) y[e] = -INFINITY;
      }
      over = fmaxf(over, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
    }
  if (__any_sync(0xffffffffu, over > kReferenceSlack || st.fresh != 0)) {
    // some row's reference moves: to the maximum of these keys, for every row that it exceeds or that has none
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t bit = 1u << (2 * rt + j);
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmaxf(top, fmaxf(x[u][rt][j], x[u][rt][2 + j]));
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float step = fmaxf(top, 0.f), keep = exp2_approx(-step);
        if (st.fresh & bit) {  // reference 0 so far, and nothing summed
          step = top == -INFINITY ? 0.f : top;
          keep = 1.f;
          if (top > -INFINITY) st.fresh &= ~bit;
        }
        st.m[rt][j] += step;
        st.l[rt][j] *= keep;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
          st.o[s][rt][j] *= keep;
          st.o[s][rt][2 + j] *= keep;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u][rt][j] -= step;
          x[u][rt][2 + j] -= step;
        }
      }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float inverse[2] = {1.f, 1.f};
    bool tiny[2] = {false, false}, some_tiny = false;
    if (kScaled && !kFine) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        tiny[h] = fabsf(keys[u].scale[h]) < kTinyScale;
        inverse[h] = tiny[h] ? 0.f : reciprocal_approx(keys[u].scale[h]);
      }
      some_tiny = __any_sync(0xffffffffu, tiny[0] || tiny[1]);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float(&y)[4] = x[u][rt];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = exp2_approx(y[e]);
      if (kFine) {
        st.l[rt][0] += y[0] + y[2];
        st.l[rt][1] += y[1] + y[3];
      }
      if (some_tiny) {
#pragma unroll
        for (int e = 0; e < 4; ++e) st.l[rt][e & 1] += tiny[e >> 1] ? y[e] : 0.f;
      }
      if (kScaled) {
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= keys[u].scale[e >> 1];
      }
      const uint32_t b0 = pack_bf16(y[0], y[1]), b1 = pack_bf16(y[2], y[3]);
      // in one part the sum takes the weights as they are rounded, so that the result is an exact mean of value rows
      if (kFine) {
        rest[u][rt][0] = transpose_8x8(pack_bf16(y[0] - __uint_as_float(b0 << 16), y[1] - __uint_as_float(b0 & 0xffff0000u)));
        rest[u][rt][1] = transpose_8x8(pack_bf16(y[2] - __uint_as_float(b1 << 16), y[3] - __uint_as_float(b1 & 0xffff0000u)));
      } else if (kScaled) {
        st.l[rt][0] = fmaf(__uint_as_float(b0 << 16), inverse[0], st.l[rt][0]);
        st.l[rt][1] = fmaf(__uint_as_float(b0 & 0xffff0000u), inverse[0], st.l[rt][1]);
        st.l[rt][0] = fmaf(__uint_as_float(b1 << 16), inverse[1], st.l[rt][0]);
        st.l[rt][1] = fmaf(__uint_as_float(b1 & 0xffff0000u), inverse[1], st.l[rt][1]);
      } else {
        ptx::add_bf16_halves(b0, st.l[rt][0], st.l[rt][1]);
        ptx::add_bf16_halves(b1, st.l[rt][0], st.l[rt][1]);
      }
      pb[u][rt][0] = transpose_8x8(b0);
      pb[u][rt][1] = transpose_8x8(b1);
    }
  }
}

// ---------------------------------------------------------------- committed slots
// Steps of 16 U keys per warp: two groups of 16 where the registers hold their rows (bytes in flight), one elsewhere.
template <int kStorage, int DP>
__host__ __device__ constexpr int groups_per_step() {
  return DP * Codes<kStorage>::kBytes <= 64 ? 2 : 1;
}

// Called where a warp met NaN codes of e4m3 among the visible slots [begin, end), all of which every row sees: in a key they make the
// whole row NaN, in a value their element, which is looked up in the pool once more.
template <int DP, int RT>
__device__ __forceinline__ uint32_t nan_elements(const wm_pool_attn_args& a, const Piece& c, int begin, int end, int w) {
  using R = Rows<WM_E4M3, DP>;
  const int lane = threadIdx.x & 31;
  const uint8_t* mask = a.key_mask != nullptr ? a.key_mask + static_cast<long long>(c.b) * a.k_len : nullptr;
  const char* v = static_cast<const char*>(a.v) + c.b * a.v_strides[0] + c.kv_head * a.v_strides[1] + R::value_piece(lane >> 2, a.head_dim) + 4 * w;
  uint32_t codes = 0;
#pragma unroll 1
  for (int j = begin + (lane & 3); j < end; j += 4)
    if (mask == nullptr || mask[j] != 0) codes |= Codes<WM_E4M3>::nan_codes(*reinterpret_cast<const uint32_t*>(v + j * a.v_strides[2]));
  codes |= __shfl_xor_sync(0xffffffffu, codes, 1);
  return codes | __shfl_xor_sync(0xffffffffu, codes, 2);
}
template <int DP, int RT>
__device__ __forceinline__ void nan_keys(const wm_pool_attn_args& a, const Piece& c, int begin, int end, bool in_key, State<DP, RT>& st) {
  const float nan = __uint_as_float(0x7fffffffu);
  if (in_key) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) st.l[rt][0] = st.l[rt][1] = nan;
  }
#pragma unroll
  for (int w = 0; w < Rows<WM_E4M3, DP>::kValueWords; ++w) {
    const uint32_t codes = nan_elements<DP, RT>(a, c, begin, end, w);
#pragma unroll
    for (int n = 0; n < 4; ++n)  // element 4 w + n of the lane's piece
      if (codes >> (8 * n + 7) & 1u) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int j = 0; j < 2; ++j) st.o[2 * w + (n >> 1)][rt][2 * (n & 1) + j] = nan;
      }
  }
}

// This warp's rows of the tiles [tile, stop) that lie among the visible slots.  With kDense the rows of the pool are DP
// elements and lie one behind the other (scales too): a lane then needs one address for all of its rows of a step.
template <int kStorage, int DP, int RT, bool kDense, bool kFine>
__device__ __forceinline__ void past_keys(const wm_pool_attn_args& a, const Piece& c, int tile, int stop, const Queries<DP, RT>& q, State<DP, RT>& st) {
  using R = Rows<kStorage, DP>;
  constexpr bool kScaled = kStorage != WM_BF16;
  constexpr int U = groups_per_step<kStorage, DP>(), kGroup = 16 * U, kStepKeys = kGroup * kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int row_bytes = kDense ? DP * R::kBytes : a.head_dim * R::kBytes;
  const float factor = a.scale * kLog2e;

  int j0 = tile * kTileKeys + warp * kGroup;
  const int end = min(c.slots, stop * kTileKeys);
  if (j0 >= end) return;
  const uint32_t k_row = kDense ? DP * R::kBytes : static_cast<uint32_t>(a.k_strides[2]) * R::kBytes;
  const uint32_t v_row = kDense ? DP * R::kBytes : static_cast<uint32_t>(a.v_strides[2]) * R::kBytes;
  const uint32_t ks_row = kDense ? 1 : static_cast<uint32_t>(a.k_scale_strides[2]), vs_row = kDense ? 1 : static_cast<uint32_t>(a.v_scale_strides[2]);
  // This lane's part of slot j0: its keys lie g, its values 2t rows on.  The launch refuses pools whose 32 rows would not
  // fit 32-bit offsets.
  const char* k = static_cast<const char*>(a.k) + (c.b * a.k_strides[0] + c.kv_head * a.k_strides[1] + j0 * a.k_strides[2]) * R::kBytes + R::key_piece(t, row_bytes);
  const char* v = static_cast<const char*>(a.v) + (c.b * a.v_strides[0] + c.kv_head * a.v_strides[1] + j0 * a.v_strides[2]) * R::kBytes + R::value_piece(g, row_bytes);
  const float* ks = kScaled ? a.k_scales + c.b * a.k_scale_strides[0] + c.kv_head * a.k_scale_strides[1] + j0 * a.k_scale_strides[2] : nullptr;
  const float* vs = kScaled ? a.v_scales + c.b * a.v_scale_strides[0] + c.kv_head * a.v_scale_strides[1] + j0 * a.v_scale_strides[2] : nullptr;
  k += g * k_row;
  v += 2 * t * v_row;
  ks += kScaled ? g * ks_row : 0;
  vs += kScaled ? g * vs_row : 0;
  const uint8_t* mask = a.key_mask != nullptr ? a.key_mask + static_cast<long long>(c.b) * a.k_len : nullptr;

  uint32_t kr[U][2][R::kKeyWords], vr[U][4][R::kValueWords];
  float kscale[U][2], vscale[U][2];
  bool open = true;  // the mask keeps slot `lane` of the step

  // Rows behind the last visible slot are not read: the last one takes their place, with weight zero.
  const auto load_k = [&](int j) {
    const int last = c.slots - 1 - j;
    if (last >= kGroup - 1) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          R::load_key(kr[u][h], k + (16 * u + 8 * h) * k_row);
          if (kScaled) {
            kscale[u][h] = ks[(16 * u + 8 * h) * ks_row];
            vscale[u][h] = vs[(16 * u + 8 * h) * vs_row];
          }
        }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int in = min(16 * u + 8 * h, last - g);  // may be negative: rows before this lane's first
          R::load_key(kr[u][h], k + in * static_cast<int>(k_row));
          if (kScaled) {
            kscale[u][h] = ks[in * static_cast<int>(ks_row)];
            vscale[u][h] = vs[in * static_cast<int>(vs_row)];
          }
        }
    }
    if (mask != nullptr) open = lane <= min(last, kGroup - 1) && mask[j + lane] != 0;
  };
  const auto load_v = [&](int j) {
    const int last = c.slots - 1 - j;
    if (last >= kGroup - 1) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 4; ++h) R::load_value(vr[u][h], v + (16 * u + (h & 1) + (h & 2) * 4) * v_row);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 4; ++h) R::load_value(vr[u][h], v + min(16 * u + (h & 1) + (h & 2) * 4, last - 2 * t) * static_cast<int>(v_row));
    }
  };

  uint32_t top_key = 0, top_value = 0;
  load_k(j0);
  load_v(j0);
  for (;;) {
    const int next = j0 + kStepKeys, room = c.slots - j0;
    constexpr uint32_t kFull = U == 2 ? 0xffffffffu : 0xffffu;
    uint32_t word = room >= kGroup ? kFull : (1u << room) - 1u;
    if (mask != nullptr) word = __ballot_sync(0xffffffffu, open);
    Keys keys[U];
    uint32_t seen[U][1][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      keys[u].all = word == kFull;
      seen[u][0][0] = seen[u][0][1] = keys[u].all ? 3u : (word >> (16 * u + g) & 1u) | (word >> (16 * u + g + 8) & 1u) << 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        keys[u].factor[h] = kScaled ? factor * kscale[u][h] : factor;
        keys[u].scale[h] = kScaled ? usable_scale(vscale[u][h], keys[u].all || (seen[u][0][0] >> h & 1u)) : 1.f;
      }
    }
    if (kStorage == WM_E4M3 && word != kFull) {  // a masked slot may hold NaN codes
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (!(seen[u][0][0] >> h & 1u)) {
#pragma unroll
            for (int w = 0; w < R::kKeyWords; ++w) kr[u][h][w] = 0;
          }
    }
    float x[U][RT][4];
#pragma unroll
    for (int u = 0; u < U; ++u) scores<kStorage, DP, RT, false>(kr[u], q, x[u], top_key);
    if (next < end) {
      k += kStepKeys * k_row;
      if (kScaled) {
        ks += kStepKeys * ks_row;
        vs += kStepKeys * vs_row;
      }
      load_k(next);
    }
    uint32_t pb[U][RT][2], rest[U][RT][2];
    weights<DP, RT, U, kScaled, false, kFine>(st, x, keys, seen, pb, rest);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!keys[u].all) {  // what a masked slot holds must not meet its zero weight
#pragma unroll
        for (int h = 0; h < 4; ++h)
          if (!(word >> (16 * u + 2 * t + (h & 1) + (h & 2) * 4) & 1u)) {
#pragma unroll
            for (int w = 0; w < R::kValueWords; ++w) vr[u][h][w] = 0;
          }
      }
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        uint32_t va[4];
        R::value_fragment(va, vr[u], s, top_value);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          mma_16816(st.o[s][rt], va[0], va[1], va[2], va[3], pb[u][rt][0], pb[u][rt][1]);
          if (kFine) mma_16816(st.o[s][rt], va[0], va[1], va[2], va[3], rest[u][rt][0], rest[u][rt][1]);
        }
      }
    }
    if (next >= end) break;
    v += kStepKeys * v_row;
    load_v(next);
    j0 = next;
  }
  if (kStorage == WM_E4M3 && __any_sync(0xffffffffu, Codes<kStorage>::some_nan(__vmaxu2(top_key, top_value))))
    nan_keys<DP, RT>(a, c, tile * kTileKeys, end, __any_sync(0xffffffffu, Codes<kStorage>::some_nan(top_key)), st);
}

// ---------------------------------------------------------------- drafted tokens
template <int kStorage, int DP, int RT, bool kFine>
__device__ __forceinline__ void draft_keys(const wm_pool_attn_args& a, const Plan& plan, const Piece& c, int tile, int stop, const Queries<DP, RT>& q, State<DP, RT>& st) {
  using R = Rows<WM_BF16, DP>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int row_bytes = a.head_dim * 2, nodes = a.q_len, words = (nodes + 31) / 32;
  const char* k = static_cast<const char*>(a.draft_k) + (c.b * a.draft_k_strides[0] + c.kv_head * a.draft_k_strides[1]) * 2 + R::key_piece(t, row_bytes);
  const char* v = static_cast<const char*>(a.draft_v) + (c.b * a.draft_v_strides[0] + c.kv_head * a.draft_v_strides[1]) * 2 + R::value_piece(g, row_bytes);
  const long long tree = a.shared_tree ? 0 : static_cast<long long>(c.b) * nodes;
  const float factor = a.scale * kLog2e;
#pragma unroll 1
  for (int i = 0; i < (stop - tile) * 2; ++i) {
    const int j0 = (tile + (i >> 1)) * kTileKeys + (i & 1) * 16 * kWarps + warp * 16;
    if (j0 >= nodes) break;
    uint32_t kr[2][R::kKeyWords], vr[4][R::kValueWords];
#pragma unroll
    for (int h = 0; h < 2; ++h) R::load_key(kr[h], k + min(j0 + g + 8 * h, nodes - 1) * a.draft_k_strides[2] * 2);
#pragma unroll
    for (int h = 0; h < 4; ++h) R::load_value(vr[h], v + min(j0 + 2 * t + (h & 1) + (h & 2) * 4, nodes - 1) * a.draft_v_strides[2] * 2);
    const bool real = lane < 16 && j0 + lane < nodes && a.depths[tree + j0 + lane] >= 0;
    const uint32_t usable = __ballot_sync(0xffffffffu, real);  // padding nodes may hold anything
    uint32_t special = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h)
#pragma unroll
      for (int w = 0; w < R::kValueWords; ++w) {
        if (!(usable >> (2 * t + (h & 1) + (h & 2) * 4) & 1u)) vr[h][w] = 0;
        special |= (vr[h][w] & 0x7f80u) == 0x7f80u || (vr[h][w] & 0x7f800000u) == 0x7f800000u;
      }
    special = __any_sync(0xffffffffu, special);
    float x[1][RT][4];
    uint32_t none = 0;
    scores<WM_BF16, DP, RT, kStorage != WM_BF16>(kr, q, x[0], none);
    uint32_t pb[1][RT][2], rest[1][RT][2], sees[RT][2], seen[1][RT][2];
    const Keys keys[1] = {{{factor, factor}, {1.f, 1.f}, false}};
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        int token, head;
        row_place(a, plan, c.kv_head, c.row_block, rt * 8 + 2 * t + j, token, head);
        sees[rt][j] = token < nodes ? a.ancestors[(tree + token) * words + (j0 >> 5)] >> (j0 & 31) & usable : 0u;
        seen[0][rt][j] = (sees[rt][j] >> g & 1u) | (sees[rt][j] >> (g + 8) & 1u) << 1;
      }
    }
    weights<DP, RT, 1, false, true, kFine>(st, x, keys, seen, pb, rest);
    if (!special) {
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        uint32_t va[4];
        R::value_fragment(va, vr, s, none);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          mma_16816(st.o[s][rt], va[0], va[1], va[2], va[3], pb[0][rt][0], pb[0][rt][1]);
          if (kFine) mma_16816(st.o[s][rt], va[0], va[1], va[2], va[3], rest[0][rt][0], rest[0][rt][1]);
        }
      }
    } else {  // an infinity or NaN among the values reaches the rows that see it and no others: row by row
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll 1
        for (int r = 0; r < 8; ++r) {
          const uint32_t row_sees = __shfl_sync(0xffffffffu, r & 1 ? sees[rt][1] : sees[rt][0], r >> 1);
          uint32_t keep[4];
#pragma unroll
          for (int h = 0; h < 4; ++h) keep[h] = 0u - (row_sees >> (2 * t + (h & 1) + (h & 2) * 4) & 1u);
          const uint32_t b0 = g == r ? pb[0][rt][0] : 0u, b1 = g == r ? pb[0][rt][1] : 0u;
#pragma unroll
          for (int s = 0; s < DP / 16; ++s) {
            uint32_t va[4], one[4][R::kValueWords];
#pragma unroll
            for (int h = 0; h < 4; ++h) one[h][s] = vr[h][s] & keep[h];
            R::value_fragment(va, one, s, none);
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            if (kFine) {
              mma_16816(x, va[0], va[1], va[2], va[3], g == r ? rest[0][rt][0] : 0u, g == r ? rest[0][rt][1] : 0u);
              // an infinity's weight may have nothing left for its second part, or have it with the other sign: the first part decides
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = fabsf(x[e]) < INFINITY ? x[e] : 0.f;
            }
            mma_16816(x, va[0], va[1], va[2], va[3], b0, b1);
            // the other columns hold 0 * infinity: only this row's is taken
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[s][rt][e] += 2 * t + (e & 1) == r ? x[e] : 0.f;
          }
        }
    }
  }
}

// ---------------------------------------------------------------- kernel
// Blocks of 128 threads that fit an SM together, from the registers that the accumulators, the rows in flight and the
// queries take; the launch holds the compiler to it, and the grid is one wave of them.
__host__ __device__ constexpr int resident_blocks(int storage, int row_tiles, int padded_dim) {
  return padded_dim > 64 ? (row_tiles == 1 || storage != WM_BF16 ? 3 : 2) : (row_tiles == 1 ? 4 : 3);
}

// How the blocks of a launch share the work.
enum Mode {
  kShares,       // equal shares of all tiles, any strides
  kDenseShares,  // the same, for pools whose rows are DP elements and lie one behind the other
  kCluster       // few short segments: one cluster per segment, which joins its blocks' sums through shared memory
};
constexpr int kMaxCluster = 8;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_blocks() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 load_remote(const void* mine, uint32_t rank) {
  float2 y;
  asm volatile("{.reg .u32 at;\nmapa.shared::cluster.u32 at, %2, %3;\nld.shared::cluster.v2.f32 {%0, %1}, [at];}"
               : "=f"(y.x), "=f"(y.y)
               : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank)
               : "memory");
  return y;
}

// The cluster's segment, cut into equal runs of tiles.
__device__ __forceinline__ Piece cluster_piece(const wm_pool_attn_args& a, const Plan& p) {
  const int n = cluster_blocks(), rank = cluster_rank(), at = blockIdx.x / n;
  Piece c;
  c.row_block = at % p.row_blocks;
  c.kv_head = at / p.row_blocks % a.kv_heads;
  c.b = at / p.row_blocks / a.kv_heads;
  c.slots = visible_slots(a, c.b);
  c.past_tiles = (c.slots + kTileKeys - 1) / kTileKeys;
  c.tiles = max(c.past_tiles + p.draft_tiles, 1);
  c.tile = c.tiles * rank / n;
  c.stop = c.tiles * (rank + 1) / n;
  c.end = 0;
  return c;
}

template <int kStorage, int DP, int RT, bool kTree, Mode kMode>
__global__ void __launch_bounds__(kThreads, resident_blocks(kStorage, RT, DP)) pool_attn_mma_kernel(const wm_pool_attn_args a, const Plan plan) {
  constexpr int kRows = RT * 8, kPitch = DP + 4;
  constexpr bool kFine = kStorage != WM_BF16;
  __shared__ __align__(16) float sm_acc[kWarps][kRows][kPitch];
  __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows];
  __shared__ uint2 sm_q[Queries<DP, RT>::kShared ? RT * (DP / 16) * 32 : 1];
  __shared__ float2 sm_sum[kMode == kCluster ? kRows : 1];  // reference and sum of the block's rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  Share share = {0, 0, 1, 0, 0};
  if (kMode != kCluster) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the joining kernel may take its place: it waits for this one's end
    share = find_share(a, plan, blockIdx.x, gridDim.x);
    if (threadIdx.x == 0) note_of(a, blockIdx.x)->last = -1;
  }
  for (int at = share.begin; at < share.end;) {
    const Piece c = kMode == kCluster ? cluster_piece(a, plan) : next_piece(a, plan, at, share.end, share.b, share.b_begin);
    at = kMode == kCluster ? 1 : c.end;
    if (kMode != kCluster && c.tile >= c.stop) continue;

    Queries<DP, RT> q;
    q.shared = sm_q;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      int token, head;
      row_place(a, plan, c.kv_head, c.row_block, rt * 8 + g, token, head);
      const bool live = token < a.q_len;
      const char* row = static_cast<const char*>(a.q) + (live ? (c.b * a.q_strides[0] + head * a.q_strides[1] + token * a.q_strides[2]) * 2 : 0);
#pragma unroll
      for (int s = 0; s < DP / 16; ++s) {
        if (Queries<DP, RT>::kShared && ((rt * (DP / 16) + s) % kWarps) != warp) continue;
        const int e = Rows<WM_BF16, DP>::key_piece(t, a.head_dim * 2) / 2 + 4 * s;
        uint2 x = make_uint2(0, 0);
        if (live && e >= t * (DP / 4)) x = *reinterpret_cast<const uint2*>(row + 2 * e);
        if (kStorage != WM_BF16) x = make_uint2(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632));
        if (Queries<DP, RT>::kShared)
          sm_q[(rt * (DP / 16) + s) * 32 + lane] = x;
        else
          q.reg[Queries<DP, RT>::kShared ? 0 : rt][Queries<DP, RT>::kShared ? 0 : s] = x;
      }
    }
    State<DP, RT> st;
    st.fresh = (1u << (2 * RT)) - 1u;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) st.m[rt][j] = 0.f, st.l[rt][j] = 0.f;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) st.o[s][rt][e] = 0.f;
    }
    if (Queries<DP, RT>::kShared) __syncthreads();

    if (c.tile < c.past_tiles) past_keys<kStorage, DP, RT, kMode == kDenseShares, kFine>(a, c, c.tile, min(c.stop, c.past_tiles), q, st);
    if (kTree && c.stop > c.past_tiles && c.stop > c.tile)
      draft_keys<kStorage, DP, RT, kFine>(a, plan, c, max(c.tile - c.past_tiles, 0), c.stop - c.past_tiles, q, st);

    // join the warps: references, sums and accumulators side by side
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = st.l[rt][j];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (st.fresh >> (2 * rt + j) & 1u) st.m[rt][j] = kNoReference;
        if (g == 0) {
          sm_m[warp][rt * 8 + 2 * t + j] = st.m[rt][j];
          sm_l[warp][rt * 8 + 2 * t + j] = l;
        }
      }
    const int d0 = Rows<WM_BF16, DP>::value_piece(g, a.head_dim * 2) / 2;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int s = 0; s < DP / 16; ++s)
          if (d0 + 2 * s >= g * (DP / 8))  // else a lower lane's
            *reinterpret_cast<float2*>(&sm_acc[warp][rt * 8 + 2 * t + j][d0 + 2 * s]) = make_float2(st.o[s][rt][j], st.o[s][rt][2 + j]);
    __syncthreads();

    // one row per thread group
    constexpr int kPerRow = kRows < kThreads ? kThreads / kRows : 1;
    const int r = threadIdx.x / kPerRow;
    int token, head;
    row_place(a, plan, c.kv_head, c.row_block, r, token, head);
    if (token < a.q_len) {
      float top = sm_m[0][r], l = 0.f, f[kWarps];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm_m[w][r]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        f[w] = exp2_approx(sm_m[w][r] - top);
        l = fmaf(sm_l[w][r], f[w], l);
      }
      bool empty = l == 0.f;
      if (kTree && a.depths[(a.shared_tree ? 0ll : static_cast<long long>(c.b) * a.q_len) + token] < 0) empty = true;  // a padding node sees nothing
      const float inverse = 1.f / l;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + c.b * a.out_strides[0] + head * a.out_strides[1] + token * a.out_strides[2];
      float* partial = kMode == kCluster ? nullptr : partial_row(a, plan, gridDim.x, blockIdx.x, c.tile == 0, r);
      if (threadIdx.x % kPerRow == 0) {
        const float2 sum = make_float2(top, empty ? 0.f : l);
        if (kMode == kCluster)
          sm_sum[r] = sum;
        else if (!whole(c))
          *reinterpret_cast<float2*>(partial) = sum;
      }
      for (int d = 2 * (threadIdx.x % kPerRow); d < a.head_dim; d += 2 * kPerRow) {
        float2 y = *reinterpret_cast<const float2*>(&sm_acc[0][r][d]);
        y.x *= f[0], y.y *= f[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
          const float2 z = *reinterpret_cast<const float2*>(&sm_acc[w][r][d]);
          y.x = fmaf(z.x, f[w], y.x);
          y.y = fmaf(z.y, f[w], y.y);
        }
        if (empty) y = make_float2(0.f, 0.f);
        if (kMode == kCluster)
          *reinterpret_cast<float2*>(&sm_acc[0][r][d]) = y;  // its own place: no other thread has read or will write it
        else if (whole(c))
          *reinterpret_cast<uint32_t*>(out + d) = empty ? 0u : pack_bf16(y.x * inverse, y.y * inverse);
        else
          *reinterpret_cast<float2*>(partial + 2 + d) = y;
      }
    }
    if constexpr (kMode != kCluster) {
      if (threadIdx.x == 0) leave_note(a, share, c, blockIdx.x, gridDim.x);
      __syncthreads();
    } else {
      // every block finishes its part of the outputs from all blocks' sums
      cluster_sync();
      const int n = cluster_blocks(), pairs = a.head_dim / 2;
      for (int i = cluster_rank() * kThreads + threadIdx.x; i < kRows * pairs; i += n * kThreads) {
        const int row = i / pairs, d = 2 * (i - row * pairs);
        row_place(a, plan, c.kv_head, c.row_block, row, token, head);
        if (token >= a.q_len) continue;
        float2 sum[kMaxCluster], y[kMaxCluster];
        float top = kNoReference, l = 0.f;
#pragma unroll
        for (int o = 0; o < kMaxCluster; ++o) {
          sum[o] = make_float2(kNoReference, 0.f);
          y[o] = make_float2(0.f, 0.f);
          if (o < n) {
            sum[o] = load_remote(&sm_sum[row], o);
            y[o] = load_remote(&sm_acc[0][row][d], o);
          }
          top = fmaxf(top, sum[o].x);
        }
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int o = 0; o < kMaxCluster; ++o) {
          const float f = exp2_approx(sum[o].x - top);
          l = fmaf(sum[o].y, f, l);
          acc.x = fmaf(y[o].x, f, acc.x);
          acc.y = fmaf(y[o].y, f, acc.y);
        }
        const float inverse = 1.f / l;
        const long long place = c.b * a.out_strides[0] + head * a.out_strides[1] + token * a.out_strides[2] + d;
        *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + place) = l == 0.f ? 0u : pack_bf16(acc.x * inverse, acc.y * inverse);
      }
      cluster_sync();  // no block leaves while another reads its shared memory
    }
  }
}

template <int kStorage, int DP, int RT, bool kTree>
cudaError_t launch_mma(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {
  if (plan.cluster > 0) {
    cudaLaunchAttribute dim = {};
    dim.id = cudaLaunchAttributeClusterDimension;
    dim.val.clusterDim.x = plan.cluster;
    dim.val.clusterDim.y = dim.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(plan.blocks);
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    config.attrs = &dim;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, pool_attn_mma_kernel<kStorage, DP, RT, kTree, kCluster>, a, plan);
  }
  // heads of 64 and 128, the usual pool: 122 us against 133 us on 64 sequences of up to 8192 int8 rows of 64, 130 us against 135 us on rows of
  // 128; rows of 96 take 139 us this way and 113 us without, rows of 32 would gain (87 against 98 us)
  if constexpr (DP % 64 == 0) {
    const bool scaled = kStorage != WM_BF16;
    if (a.head_dim == DP && a.k_strides[2] == DP && a.v_strides[2] == DP && (!scaled || (a.k_scale_strides[2] == 1 && a.v_scale_strides[2] == 1))) {
      pool_attn_mma_kernel<kStorage, DP, RT, kTree, kDenseShares><<<plan.blocks, kThreads, 0, stream>>>(a, plan);
      return cudaGetLastError();
    }
  }
  pool_attn_mma_kernel<kStorage, DP, RT, kTree, kShares><<<plan.blocks, kThreads, 0, stream>>>(a, plan);
  return cudaGetLastError();
}

template <int kStorage, int DP, bool kTree>
cudaError_t launch_mma_rows(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {
  switch (plan.rows_per_block) {
    case 8: return launch_mma<kStorage, DP, 1, kTree>(a, plan, stream);
    case 16: return launch_mma<kStorage, DP, 2, kTree>(a, plan, stream);
  }
  return cudaErrorInvalidValue;  // not reached: more than 16 rows go through shared memory (pool_attn_shared.cuh)
}

// One translation unit per way of holding the pool, with and without drafted tokens.
template <int kStorage, bool kTree>
cudaError_t launch_mma_storage(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream);

#define WM_POOL_ATTN_UNIT(kStorage, kTree)                                                                                          \
  template <>                                                                                                                       \
  cudaError_t launch_mma_storage<kStorage, kTree>(const wm_pool_attn_args& a, const Plan& plan, cudaStream_t stream) {              \
    if (a.head_dim <= 32) return launch_mma_rows<kStorage, 32, kTree>(a, plan, stream);                                             \
    if (a.head_dim <= 64) return launch_mma_rows<kStorage, 64, kTree>(a, plan, stream);                                             \
    if (a.head_dim <= 96) return launch_mma_rows<kStorage, 96, kTree>(a, plan, stream);                                             \
    return launch_mma_rows<kStorage, 128, kTree>(a, plan, stream);                                                                  \
  }

}  // namespace pool
}  // namespace wm
