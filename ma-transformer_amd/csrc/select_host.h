// select_host.h -- what the two units behind ma_select.h share on the host.
#pragma once

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "host_common.h"
#include "ma_attn.h"
#include "ma_select.h"

namespace ma_select_host {

using ma_host::fail;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The kernels' bitmaps of one chunk hold a word per block in LDS.
constexpr int64_t kMaxBlocks = 16384;

inline int64_t blocks_of(const ma_select_desc* d) { return (d->seq_len + d->block_size - 1) / d->block_size; }

inline int check(const ma_select_desc* d, const char* who) {
  if (!d) return fail("%s: null descriptor", who);
  if (d->dtype != MA_ATTN_F32 && d->dtype != MA_ATTN_BF16 && d->dtype != MA_ATTN_F16)
    return fail("%s: unsupported dtype %d", who, d->dtype);
  if (d->batch < 0 || d->seq_len < 0) return fail("%s: negative size", who);
  if (d->num_kv_heads < 1 || d->num_heads < 1 || d->num_heads % d->num_kv_heads)
    return fail("%s: num_heads (%lld) must be a multiple of num_kv_heads (%lld)", who, (long long)d->num_heads,
                (long long)d->num_kv_heads);
  if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8)
    return fail("%s: head_dim must be a multiple of 8 from 8 to 128, got %lld", who, (long long)d->head_dim);
  if (d->block_size != 16 && d->block_size != 32 && d->block_size != 64)
    return fail("%s: block_size must be 16, 32 or 64, got %lld", who, (long long)d->block_size);
  if (d->num_selected < 1 || d->num_selected > 64)
    return fail("%s: num_selected must be in [1, 64], got %lld", who, (long long)d->num_selected);
  if (d->num_heads > (1 << 16)) return fail("%s: too many heads", who);
  if (d->seq_len > kMaxBlocks * d->block_size)
    return fail("%s: at most %lld blocks a sequence", who, (long long)kMaxBlocks);
  if (d->batch > (INT32_MAX >> 8) || (d->batch > 0 && d->seq_len > ((int64_t)1 << 40) / (d->batch * d->num_heads)))
    return fail("%s: batch * seq_len * heads too large", who);
  return 0;
}

inline int check_aligned(std::initializer_list<const void*> ps, const char* who) {
  for (const void* p : ps) {
    if (!p) return fail("%s: null pointer", who);
    if (!aligned16(p)) return fail("%s: tensors must be 16-byte aligned", who);
  }
  return 0;
}

struct Events {
  explicit Events(const ma_select_desc* d) {
    ma_host::g_ev_start = static_cast<hipEvent_t>(d->start_event);
    ma_host::g_ev_stop = static_cast<hipEvent_t>(d->stop_event);
  }
  ~Events() { ma_host::g_ev_start = ma_host::g_ev_stop = nullptr; }
};

inline int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: kernel launch failed: %s", who, hipGetErrorString(e));
}

}  // namespace ma_select_host
