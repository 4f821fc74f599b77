/*
 * mingpaged.h — C ABI of the paged cache in libmingmoe.so: several streams' keys and values held in pages of one pool,
 * the append of new tokens with their position rotation, and the attentions of new tokens (one per stream in decode, a
 * piece or the whole of a prompt) on MI355X (gfx950).
 *
 * The conventions are those of mingmoe.h: device pointers, strides in elements, dtype codes, a hipStream_t as void*, an
 * int status with mm_last_error()'s message; nothing allocates, frees or synchronises, every call can be captured.
 *
 * The reference has no batch of streams: its caches are static ones of a single stream (StaticQwen2, engine.py:1258-1259,
 * and StaticHybridCache, engine.py:537-548), and its attentions those that mm_qwen_decode_attn, mm_mla_decode_attn and
 * mm_mla_prefill_attn replace. A contiguous cache [heads, max_len, d] of such a stream is one page of max_len rows here.
 */
#ifndef MINGPAGED_H
#define MINGPAGED_H

#include <stddef.h>
#include <stdint.h>

#include "mingmoe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MM_PAGED_VERSION 2

/* The pool: k [n_pages, nkv, page, dqk] and v [n_pages, nkv, page, dv] of dtype (MM_BF16 / MM_FP16), any strides of the
 * first three dims (multiples of 8; so [n_pages, page, nkv, d] pools are strides too), the last one contiguous, 16-byte
 * aligned. dqk, dv: multiples of 8 up to 256. */
typedef struct mm_pages {
  void* k;
  void* v;
  int32_t dtype;
  int32_t nkv;
  int32_t dqk;
  int32_t dv;
  int64_t n_pages;
  int64_t page; /* rows (positions) of a page, any number >= 1 */
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
} mm_pages;

/* A batch of packed tokens. Stream b owns tokens cu[b] .. cu[b+1] - 1 (n_b of them; 0 is allowed); kv_lens[b] rows of its
 * cache count, its new tokens' among them, so its token i stands at position kv_lens[b] - n_b + i. Position p of stream b
 * is row p % page of page table[b * table_stride + p / page]. cu [seqs + 1], kv_lens [seqs] and table [seqs, max_pages]
 * are device arrays of one dtype (idx_dtype: MM_INT32 / MM_INT64), read when the call runs: one captured graph serves
 * every length. cu starts at 0, does not fall and ends at or below `tokens`; rows of the outputs behind its end are left
 * as they were. */
typedef struct mm_batch {
  const void* cu;
  const void* kv_lens;
  const void* table;
  int64_t table_stride;
  int64_t max_pages;
  int64_t seqs;
  int64_t tokens;
  int32_t idx_dtype;
} mm_batch;

/* Rows [tokens, heads, d] of a packed tensor: strides in elements (multiples of 8; those of a dim of one are not used), the
 * last dim contiguous, rows 16-byte aligned (of an attention's output 8-byte, strides multiples of 4). */
typedef struct mm_rows {
  void* p;
  int64_t token_stride;
  int64_t head_stride;
} mm_rows;

/* MM_PAGED_VERSION of the library. */
int mm_paged_version(void);

/* The new tokens' keys and values into their pages, rotated on the way: q, k [tokens, nh / nkv, dqk] and v [tokens, nkv,
 * dv] of pages.dtype. Dims rot_offset .. rot_offset + 2 * pairs - 1 of every q and k head turn by position * inv_freq[j]
 * (inv_freq fp32 [pairs] on the device; the angle is reduced in 64 bits, so far positions lose nothing): pairs (x[j],
 * x[j + pairs]) of that range, or with interleaved != 0 (x[2j], x[2j + 1]); one rounding. pairs and rot_offset multiples of
 * 8; inv_freq NULL: no rotation. The rotated q goes to q_out (may be q itself), the rotated k to its page and, where
 * k_out.p is not NULL, to k_out (may be k itself); v to its page. A position outside [0, max_pages * page), a page id
 * outside [0, n_pages), and every token of a stream whose kv_lens lies outside [0, max_pages * page] store nothing into the
 * pool; q_out and k_out are written all the same. Two streams that share a page must not append to the same rows of it. */
typedef struct mm_paged_append_args {
  mm_pages pages;
  mm_batch batch;
  mm_rows q, k, v, q_out, k_out;
  const float* inv_freq;
  int64_t pairs;
  int32_t nh;
  int32_t rot_offset;
  int32_t interleaved;
} mm_paged_append_args;
int mm_paged_append(const mm_paged_append_args* args, void* stream);

/* Bytes of workspace mm_paged_attn needs for a batch of these sizes (max_keys = max_pages * page), or with at_most != 0
 * for every batch of at most these tokens, streams and keys; 0: none, -1 if invalid. */
int64_t mm_paged_attn_workspace(int64_t tokens, int64_t seqs, int64_t max_keys, int nh, int nkv, int dqk, int dv,
                                int at_most);

/* Attention of the new tokens over the paged cache that already holds their own rows (mm_paged_append): token i of stream
 * b, at position p = kv_lens[b] - n_b + i, takes softmax(scale * q . K[0..p]^T) . V[0..p], query head h on key / value
 * head h / (nh / nkv). q [tokens, nh, dqk], out [tokens, nh, dv] of pages.dtype. Scores, statistics and sums in fp32; the
 * weights enter the value product rounded to the cache's type. Positions whose page id lies outside [0, n_pages) are left
 * out; a token with no position left gets zeros; the tokens of a stream whose kv_lens lies outside [0, max_pages * page]
 * get NaN. Rows past a token's position never reach it, whatever they hold. out must not overlap q or the pool. workspace:
 * mm_paged_attn_workspace bytes, 16-byte aligned (NULL where that is 0), no initialisation; calls that share one must not
 * overlap in time. Equal calls give equal bits; the order of a token's sums depends on the whole batch's lengths. Limits:
 * tokens 2^22, tokens * nh 2^30, streams 2^20, max_pages * page 2^30; a launch of 2^23 workgroups (blocks of 16 or 128 rows
 * times key / value heads, a stream's own each) is refused. */
typedef struct mm_paged_attn_args {
  mm_pages pages;
  mm_batch batch;
  mm_rows q, out;
  void* workspace;
  int64_t workspace_bytes;
  int32_t nh;
  float scale;
} mm_paged_attn_args;
int mm_paged_attn(const mm_paged_attn_args* args, void* stream);

/* Bytes of workspace mm_prompt_attn needs, as mm_paged_attn_workspace. */
int64_t mm_prompt_attn_workspace(int64_t tokens, int64_t seqs, int nh, int nkv, int dqk, int dv, int at_most);

/* Causal attention over whole prompts packed one behind the other: token i of prompt b (tokens cu[b] .. cu[b+1] - 1)
 * takes softmax(scale * q . K[0..i]^T) . V[0..i] over its own prompt's rows of k [tokens, nkv, dqk] and v [tokens, nkv,
 * dv]. dtype MM_BF16 / MM_FP16; rounding, rows behind the last prompt, limits and workspace as for mm_paged_attn; cu
 * [seqs + 1] of idx_dtype on the device. */
typedef struct mm_prompt_attn_args {
  mm_rows q, k, v, out;
  const void* cu;
  int64_t seqs;
  int64_t tokens;
  void* workspace;
  int64_t workspace_bytes;
  int32_t idx_dtype;
  int32_t dtype;
  int32_t nh;
  int32_t nkv;
  int32_t dqk;
  int32_t dv;
  float scale;
} mm_prompt_attn_args;
int mm_prompt_attn(const mm_prompt_attn_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MINGPAGED_H */
