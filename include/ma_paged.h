/*
 * ma_paged.h -- C-ABI of the paged key/value cache (libma_attn.so): serving
 * one new token at a time.
 *
 * A cache holds `num_pages` pages of `page_size` tokens each, keys and values
 * [num_pages, page_size, num_kv_heads, head_dim] in one dtype.  Stream b's
 * token t lies in page page_table[b, t / page_size], slot t % page_size.
 * Query head h reads key/value head h / (num_heads / num_kv_heads).
 *
 * The functions return 0, or non-zero with a message in ma_attn_last_error().
 * They allocate nothing, never synchronise, and are asynchronous on `stream`
 * (hipStream_t).  Page tables, lengths and page lists are read on the device:
 * entries outside their range are skipped (never followed), lengths are
 * clamped to the table.
 */
#ifndef MA_PAGED_H
#define MA_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ma_paged_desc {
  int64_t batch;
  int64_t num_tokens;   /* append: new tokens per stream (rows of key/value/query) */
  int64_t num_heads;    /* query heads, a multiple of num_kv_heads */
  int64_t num_kv_heads;
  int64_t head_dim;     /* a multiple of 8, at most 128 */
  int64_t num_pages;
  int64_t page_size;    /* a multiple of 16 */
  int64_t table_width;  /* page_table is int32 [batch, table_width] */
  int32_t dtype;        /* MA_ATTN_F32, MA_ATTN_BF16, MA_ATTN_F16 */
  int32_t interleaved;  /* append: rotate (2j, 2j+1) instead of (j, j + rotary_dim/2) */
  int64_t rotary_dim;   /* append: 0 (none) or a multiple of 16, at most head_dim */
  int64_t left;         /* decode: keys [len-1-left, len-1]; negative: all */
  int64_t num_global;   /* decode: with left >= 0, also the keys [0, num_global) */
  int64_t num_selected; /* decode: entries per (stream, kv head) of `pages`; select: entries to list */
  int64_t first_pages;  /* select: this many first pages are always listed */
  int64_t local_pages;  /* select: this many newest pages are always listed (>= 1) */
  float scale;          /* decode: softmax scale; 0: 1/sqrt(head_dim) */
  int32_t reserved;
  void* start_event;    /* hipEvent_t stamped on the call's first kernel start, or NULL */
  void* stop_event;     /* hipEvent_t stamped on the call's last kernel end, or NULL */
} ma_paged_desc;

/*
 * Appends counts[b] (NULL: num_tokens) tokens of key/value
 * [batch, num_tokens, num_kv_heads, head_dim] to stream b at positions
 * start[b], start[b] + 1, ..., keys rotated by position * inv_freq[j]
 * (float64 [rotary_dim / 2]).  query (or NULL) [batch, num_tokens, num_heads,
 * head_dim] is rotated the same way into query_out (every row).
 * key_sums (or NULL), float32 [num_pages, num_kv_heads, head_dim]: the sums of
 * the stored keys of every page that receives tokens, over its slots up to the
 * last new one, are written.
 */
int ma_paged_append(const ma_paged_desc* desc, const void* key, const void* value, const void* query,
                    void* query_out, void* cache_key, void* cache_value, float* key_sums,
                    const int32_t* page_table, const int32_t* start, const int32_t* counts,
                    const double* inv_freq, void* stream);

/* Bytes of device workspace ma_paged_decode needs. */
size_t ma_paged_decode_workspace_size(const ma_paged_desc* desc);

/*
 * Attention of one query token per stream, query/out [batch, num_heads,
 * head_dim], over the lengths[b] tokens of stream b.  pages (or NULL): int32
 * [batch, num_kv_heads, num_selected] logical pages to read instead of all of
 * them; a repeated entry counts once.  lse (or NULL): float32
 * [batch, num_heads], log2 of the sum of exp(scaled scores).  A query without
 * keys gives zeros and lse -inf.
 */
int ma_paged_decode(const ma_paged_desc* desc, const void* query, const void* cache_key, const void* cache_value,
                    const int32_t* page_table, const int32_t* lengths, const int32_t* pages, void* out, float* lse,
                    void* workspace, size_t workspace_bytes, void* stream);

/*
 * Lists, per stream and key/value head, the num_selected pages with the
 * largest score (sum of the group's queries) . (page key sum / page_size),
 * computed in float64; first_pages and local_pages are always listed, ties go
 * to the lower page, NaN scores rank last.  pages: int32
 * [batch, num_kv_heads, num_selected], ascending logical pages, -1 behind them.
 */
int ma_paged_select(const ma_paged_desc* desc, const void* query, const float* key_sums, const int32_t* page_table,
                    const int32_t* lengths, int32_t* pages, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MA_PAGED_H */
