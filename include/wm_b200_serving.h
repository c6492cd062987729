/*
 * wm_b200_serving.h -- C ABI of the serving operators around the KV pool: a pool held in 8 bits (commit, read,
 * read back) and the pass over drafted tokens that branch (tree tables, tree attention).
 *
 * The conventions of wm_b200.h hold: plain device pointers, element strides, asynchronous launches on `stream`, no
 * allocation, no host synchronisation, 0 or a negative WM_E* code with the text in wm_last_error().  None of these
 * operators has a counterpart in the upstream project, whose pool is bf16 and whose decoding is one token at a time.
 *
 * An 8-bit pool holds every row of head_dim elements as codes and one fp32 scale; an element stands for code * scale:
 *   WM_INT8  scale = a / 127, code = round(x * (127 / a)), a the row's largest magnitude, both quotients and the
 *            product rounded to fp32, halves to even;
 *   WM_E4M3  scale = the smallest power of two with a / scale <= 448, code = x / scale rounded to e4m3, halves to even.
 * A row with a < 2^-100 is held as zeros with scale 0; a row with an infinity or NaN gets codes 0 and scale NaN and
 * reads back as NaN throughout.
 * In a pool that was quantised elsewhere e4m3's two NaN codes are NaN to the read back and to every query that sees them.
 */
#ifndef WM_B200_SERVING_H
#define WM_B200_SERVING_H

#include "wm_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of a pool, next to WM_F32 and WM_BF16 */
#define WM_INT8 2
#define WM_E4M3 3

/* Commit of new K and V rows to a pool at device-resident lengths, quantised on the way when the pool is held in
 * 8 bits.  Row i of sequence b goes to slot lengths[b] + lead + i, for i < rows and, with counts, i < counts[b]; it
 * is row i of the source or, with index, row index[b*rows + i] of its source_rows rows.  Slots outside the pool and
 * indices outside the source are skipped: such a slot keeps what it held.  Pool tensors are (batch, heads, slots,
 * head_dim), scales (batch, heads, slots), sources (batch, heads, source_rows, head_dim), with element strides for
 * (batch, head, token).  head_dim is a multiple of 16 up to 128; pool rows and source rows are 16-byte aligned.
 * The pool must not overlap the source.  More than 2^31 - 65536 sequences are refused. */
typedef struct wm_pool_commit_args {
  void* keys;
  void* values;
  float* key_scales; /* NULL for a WM_F32 / WM_BF16 pool */
  float* value_scales;
  const void* new_keys;
  const void* new_values;
  const void* lengths;
  const int32_t* index;  /* (batch, rows) or NULL */
  const int32_t* counts; /* (batch,) or NULL */
  int64_t key_strides[3];
  int64_t value_strides[3];
  int64_t key_scale_strides[3];
  int64_t value_scale_strides[3];
  int64_t new_key_strides[3];
  int64_t new_value_strides[3];
  int32_t storage; /* of the pool; WM_F32 / WM_BF16 only when equal to dtype */
  int32_t dtype;   /* of the new rows */
  int32_t batch, heads, slots, rows, source_rows, head_dim;
  int32_t lead; /* 1 when slot 0 is the shared dummy */
  int32_t lengths_is64;
} wm_pool_commit_args;

/* The rows an 8-bit pool stands for: out = code * scale in `dtype`; rows at or behind lengths[b] + lead are written as
 * zeros and not read (lengths NULL: every row is live).  codes (batch, heads, slots, head_dim), scales (batch, heads,
 * slots), out like codes, element strides for (batch, head, token), 16-byte aligned rows.  More than 2^31 - 65536 (sequence,
 * head) pairs are refused. */
typedef struct wm_pool_dequant_args {
  const void* codes;
  const float* scales;
  const void* lengths;
  void* out;
  int64_t code_strides[3];
  int64_t scale_strides[3];
  int64_t out_strides[3];
  int32_t storage, dtype;
  int32_t batch, heads, slots, head_dim;
  int32_t lead;
  int32_t lengths_is64;
} wm_pool_dequant_args;

/* Tables of trees of drafted tokens.  parents (batch, tokens): the node a node hangs on, -1 for the committed prefix.
 * A node whose chain of parents does not end in -1 (another negative number, a number beyond the last node, a cycle)
 * is padding.  ancestors (batch, tokens, ceil(tokens / 32)): bit j % 32 of word j / 32 of row i says that node i
 * attends to node j, an ancestor of i (or i itself with include_self); rows of padding nodes are zero.  depths
 * (batch, tokens): the number of ancestors, -1 for padding.  tokens <= 512. */
typedef struct wm_draft_tree_args {
  const int32_t* parents;
  uint32_t* ancestors;
  int32_t* depths;
  int32_t batch, tokens, include_self;
} wm_draft_tree_args;

/* Attention of q_len queries per sequence that stand behind the committed tokens of a pool: every query sees the slots
 * s < lengths[b] + lead (lengths NULL: all) that key_mask keeps.  With ancestors, the queries are the nodes of a tree of
 * drafted tokens: node i also sees the rows j of draft_k / draft_v that its ancestor bits name, and a padding node
 * (depths[i] < 0) sees nothing.  Rows that see nothing are written as zeros.  Rows of the pool that are not seen are
 * not read, or not used; rows of padding nodes in draft_k / draft_v neither.
 * head_dim at most 128, rows of every tensor multiples of 16 bytes and 16-byte aligned, at most 512 drafted tokens; rows of
 * the pool and of its scales lie less than 2^24 elements apart; batch * kv_heads * row blocks * tiles of 128 keys below 2^31.
 * Other calls are refused with WM_EUNSUPPORTED.  The workspace (wm_pool_attn_workspace_bytes, 16-byte aligned, the same for every content of the
 * tensors) must not be shared by calls that may run at once. */
typedef struct wm_pool_attn_args {
  const void* q; /* (batch, q_heads, q_len, head_dim) */
  const void* k; /* (batch, kv_heads, k_len, head_dim) in `storage` */
  const void* v;
  const float* k_scales; /* (batch, kv_heads, k_len), 8-bit pools */
  const float* v_scales;
  const void* draft_k; /* (batch, kv_heads, q_len, head_dim) in `dtype`, or NULL */
  const void* draft_v;
  const uint32_t* ancestors; /* (batch | 1, q_len, ceil(q_len / 32)), or NULL */
  const int32_t* depths;     /* (batch | 1, q_len) */
  const void* lengths;
  const uint8_t* key_mask; /* (batch, k_len) 0/1, or NULL */
  void* out;
  void* workspace;
  size_t workspace_bytes;
  int64_t q_strides[3];
  int64_t k_strides[3];
  int64_t v_strides[3];
  int64_t k_scale_strides[3];
  int64_t v_scale_strides[3];
  int64_t draft_k_strides[3];
  int64_t draft_v_strides[3];
  int64_t out_strides[3];
  int32_t dtype;   /* of q, the drafts and out: WM_F32 or WM_BF16 */
  int32_t storage; /* of k and v: dtype, WM_INT8 or WM_E4M3 */
  int32_t batch, q_heads, kv_heads, q_len, k_len, head_dim;
  int32_t lead;
  int32_t lengths_is64;
  int32_t shared_tree; /* one tree for the whole batch */
  float scale;
} wm_pool_attn_args;

WM_API size_t wm_pool_attn_workspace_bytes(const wm_pool_attn_args* args);

WM_API int wm_pool_commit(const wm_pool_commit_args* args, void* stream);

/* The lengths behind a commit, in place: lengths[b] grows by the rows that were written, to `capacity` at most.  Those are rows, with
 * counts counts[b] of them at most, with index (batch, rows) those before the first index outside the source's source_rows. */
WM_API int wm_pool_advance(void* lengths, int32_t lengths_is64, const int32_t* index, const int32_t* counts, int32_t batch,
                           int32_t rows, int32_t source_rows, int32_t capacity, void* stream);
WM_API int wm_pool_dequant(const wm_pool_dequant_args* args, void* stream);
WM_API int wm_draft_tree(const wm_draft_tree_args* args, void* stream);
WM_API int wm_pool_attn(const wm_pool_attn_args* args, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* WM_B200_SERVING_H */
