/*
 * ma_select.h -- C-ABI of block selection and of the attention over selected
 * blocks (libma_attn.so).
 *
 * Queries [batch, seq_len, num_heads, head_dim], keys and values
 * [batch, seq_len, num_kv_heads, head_dim]; query head h reads key/value head
 * h / (num_heads / num_kv_heads).  The sequence is cut into blocks of
 * `block_size` keys; `blocks` is int32 [batch, seq_len, num_kv_heads,
 * num_selected]: for each query and key/value head the blocks it attends.
 * Entries outside [0, ceil(seq_len / block_size)), repeats and, when causal,
 * blocks that begin behind the query are skipped.
 *
 * The functions return 0, or non-zero with a message in ma_attn_last_error().
 * They allocate nothing, never synchronise, and are asynchronous on `stream`.
 */
#ifndef MA_SELECT_H
#define MA_SELECT_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ma_select_desc {
  int64_t batch;
  int64_t seq_len;
  int64_t num_heads;    /* a multiple of num_kv_heads */
  int64_t num_kv_heads;
  int64_t head_dim;     /* a multiple of 8, at most 128 */
  int64_t block_size;   /* 16, 32 or 64 */
  int64_t num_selected; /* 1 to 64 */
  int32_t dtype;        /* MA_ATTN_F32, MA_ATTN_BF16, MA_ATTN_F16 */
  int32_t causal;       /* keys up to the query's own only */
  int64_t first_blocks; /* select: this many first blocks are always listed */
  int64_t local_blocks; /* select: the query's own block and the ones before it, this many, are always listed (>= 1) */
  float scale;          /* attention: softmax scale; 0: 1/sqrt(head_dim) */
  int32_t reserved;
  void* start_event;    /* hipEvent_t stamped on the call's first kernel start, or NULL */
  void* stop_event;     /* hipEvent_t stamped on the call's last kernel end, or NULL */
} ma_select_desc;

/*
 * Lists for each query and key/value head the num_selected blocks with the
 * largest score (sum of the group's queries) . (mean of the block's keys), in
 * float64; ties go to the lower block, NaN scores rank last.  blocks:
 * ascending, -1 behind them.
 */
int ma_select_blocks(const ma_select_desc* desc, const void* q, const void* k, int32_t* blocks, void* workspace,
                     size_t workspace_bytes, void* stream);
size_t ma_select_blocks_workspace_size(const ma_select_desc* desc);

/*
 * o [batch, seq_len, num_heads, head_dim]: softmax attention of each query
 * over the keys of its blocks; a query without keys gives zeros.  lse (or
 * NULL): float32 [batch, seq_len, num_heads], log2 of the sum of exp(scaled
 * scores), -inf without keys.
 */
int ma_selected_forward(const ma_select_desc* desc, const void* q, const void* k, const void* v,
                        const int32_t* blocks, void* o, float* lse, void* workspace, size_t workspace_bytes,
                        void* stream);
size_t ma_selected_forward_workspace_size(const ma_select_desc* desc);

/* dQ, dK, dV of ma_selected_forward from its output and statistics. */
int ma_selected_backward(const ma_select_desc* desc, const void* q, const void* k, const void* v,
                         const int32_t* blocks, const void* o, const float* lse, const void* dout, void* dq,
                         void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream);
size_t ma_selected_backward_workspace_size(const ma_select_desc* desc);

#ifdef __cplusplus
}
#endif

#endif /* MA_SELECT_H */
