// paged.hip -- the C-ABI of the paged cache (ma_paged.h): argument checks and
// launches of paged_kernel.h.
#include "ma_paged.h"

#include <algorithm>
#include <cmath>

#include "host_common.h"
#include "ma_attn.h"
#include "paged_kernel.h"

namespace {

using namespace ma_paged;
using ma_host::fail;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A launch holds fewer than 2^32 threads; workgroups have at most 1024.
constexpr int64_t kMaxGrid = INT32_MAX / 1024;

// What every call needs of a descriptor.
int check(const ma_paged_desc* d, const char* who) {
  if (!d) return fail("%s: null descriptor", who);
  if (d->dtype != MA_ATTN_F32 && d->dtype != MA_ATTN_BF16 && d->dtype != MA_ATTN_F16)
    return fail("%s: unsupported dtype %d", who, d->dtype);
  if (d->batch < 0 || d->num_tokens < 0 || d->num_pages < 0 || d->table_width < 0)
    return fail("%s: negative size", who);
  if (d->num_kv_heads < 1 || d->num_heads < 1 || d->num_heads % d->num_kv_heads)
    return fail("%s: num_heads (%lld) must be a multiple of num_kv_heads (%lld)", who, (long long)d->num_heads,
                (long long)d->num_kv_heads);
  if (d->head_dim < 8 || d->head_dim > 128 || d->head_dim % 8)
    return fail("%s: head_dim must be a multiple of 8 from 8 to 128, got %lld", who, (long long)d->head_dim);
  if (d->page_size < 16 || d->page_size % 16 || d->page_size > (1 << 20))
    return fail("%s: page_size must be a multiple of 16 up to 2^20, got %lld", who, (long long)d->page_size);
  if (d->num_heads > (1 << 16)) return fail("%s: too many heads", who);
  // token slots and tokens per stream are 32-bit in the kernels (bytes are not)
  if (d->num_pages > (int64_t)INT32_MAX / d->page_size || d->table_width > (int64_t)INT32_MAX / d->page_size)
    return fail("%s: num_pages * page_size and table_width * page_size must stay below 2^31 tokens", who);
  if (d->batch > INT32_MAX / (1 << 8)) return fail("%s: batch too large", who);
  return 0;
}

struct Events {
  explicit Events(const ma_paged_desc* d) {
    ma_host::g_ev_start = static_cast<hipEvent_t>(d->start_event);
    ma_host::g_ev_stop = static_cast<hipEvent_t>(d->stop_event);
  }
  ~Events() { ma_host::g_ev_start = ma_host::g_ev_stop = nullptr; }
};

int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : fail("%s: kernel launch failed: %s", who, hipGetErrorString(e));
}

// Workgroups a decode call splits its token range over: from 2048 keys on, as
// many as fill the card (1024, four a CU).  A split costs the second launch:
// 1024 listed keys of 32 x 4 heads take 11.7 us unsplit (12.4 when two parts
// were measured at 11.4 + 4.0); 65536 keys of 8 heads 24-26 us in 64 to 256 parts.  Units = (stream, kv
// head, 16 query heads).
int64_t decode_splits(const ma_paged_desc* d) {
  const int64_t G = d->num_heads / d->num_kv_heads;
  const int64_t units = d->batch * d->num_kv_heads * ((G + 15) / 16);
  int64_t keys = d->table_width * d->page_size;
  if (d->num_selected > 0)
    keys = std::min(keys, d->num_selected * d->page_size);
  else if (d->left >= 0 && d->left < keys)
    keys = std::min(keys, d->left + 32 + std::min(std::max<int64_t>(d->num_global, 0), keys));
  const int64_t most = std::max<int64_t>(1, keys / 1024);
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(units, 1));
  return std::min({most, want, (int64_t)kMaxSplit});
}

template <typename T>
int append_t(const ma_paged_desc* d, AppendArgs a, hipStream_t st) {
  const size_t angles = (size_t)kAppendTile * (size_t)(d->rotary_dim / 2) * sizeof(double2);
  const size_t shm = std::max(angles, a.sums ? (size_t)kAppendThreads * 8 * sizeof(float) : (size_t)16);
  const int64_t grid = d->batch * a.wgs;
  ma_host::launch(true, append_kernel<T>, dim3((unsigned)grid), dim3(kAppendThreads), (uint32_t)shm, st, a);
  return launched("ma_paged_append");
}

template <typename T, int DP>
void decode_dp(const DecodeArgs& a, int64_t grid, bool join, hipStream_t st) {
  if (a.D == DP)
    ma_host::launch(!join, decode_kernel<T, DP, true>, dim3((unsigned)grid), dim3(64 * kDecWaves), 0, st, a);
  else
    ma_host::launch(!join, decode_kernel<T, DP, false>, dim3((unsigned)grid), dim3(64 * kDecWaves), 0, st, a);
}

template <typename T>
int decode_t(const ma_paged_desc* d, const DecodeArgs& a, hipStream_t st) {
  const int64_t grid = d->batch * a.Hkv * a.gt * a.nsplit;
  const bool join = a.nsplit > 1;
  if (a.D <= 32)
    decode_dp<T, 32>(a, grid, join, st);
  else if (a.D <= 64)
    decode_dp<T, 64>(a, grid, join, st);
  else
    decode_dp<T, 128>(a, grid, join, st);
  const dim3 rows((unsigned)(d->batch * a.H)), threads(kJoinThreads);
  if (join && a.D <= 32)
    ma_host::launch(true, decode_join_kernel<T, 32>, rows, threads, 0, st, a);
  else if (join && a.D <= 64)
    ma_host::launch(true, decode_join_kernel<T, 64>, rows, threads, 0, st, a);
  else if (join)
    ma_host::launch(true, decode_join_kernel<T, 128>, rows, threads, 0, st, a);
  return launched("ma_paged_decode");
}

}  // namespace

extern "C" {

int ma_paged_append(const ma_paged_desc* d, const void* key, const void* value, const void* query, void* query_out,
                    void* cache_key, void* cache_value, float* key_sums, const int32_t* page_table,
                    const int32_t* start, const int32_t* counts, const double* inv_freq, void* stream) {
  ma_host::clear_error();
  const char* who = "ma_paged_append";
  if (check(d, who)) return 1;
  if (d->rotary_dim < 0 || d->rotary_dim % 16 || d->rotary_dim > d->head_dim)
    return fail("%s: rotary_dim must be a multiple of 16 up to head_dim, got %lld", who, (long long)d->rotary_dim);
  if (d->batch == 0 || d->num_tokens == 0) return 0;
  if (!key || !value || !start || (query && !query_out) || (d->rotary_dim && !inv_freq) ||
      (d->table_width && !page_table) || (d->num_pages && (!cache_key || !cache_value)))
    return fail("%s: null pointer", who);
  for (const void* p : {key, value, query, (const void*)query_out, (const void*)cache_key, (const void*)cache_value})
    if (!aligned16(p)) return fail("%s: tensors must be 16-byte aligned", who);
  if (d->num_tokens > INT32_MAX / 2) return fail("%s: num_tokens too large", who);
  AppendArgs a{};
  a.k = key;
  a.v = value;
  a.q = query;
  a.qo = query_out;
  a.ck = cache_key;
  a.cv = cache_value;
  a.sums = key_sums;
  a.table = page_table;
  a.start = start;
  a.counts = counts;
  a.freq = inv_freq;
  a.n = d->num_tokens;
  a.width = d->table_width;
  a.pages = d->num_pages;
  a.page = (int32_t)d->page_size;
  a.step = key_sums ? a.page : 64;
  a.H = (int32_t)d->num_heads;
  a.Hkv = (int32_t)d->num_kv_heads;
  a.D = (int32_t)d->head_dim;
  a.R = (int32_t)d->rotary_dim;
  a.inter = d->interleaved != 0;
  // positions start anywhere in a page, so one more than the rows alone fill
  const int64_t wgs = key_sums ? (d->num_tokens - 1 + a.step - 1) / a.step + 1 : (d->num_tokens + 63) / 64;
  if (wgs * d->batch > kMaxGrid) return fail("%s: batch * num_tokens too large", who);
  a.wgs = (int32_t)wgs;
  Events ev(d);
  (void)hipGetLastError();
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->dtype == MA_ATTN_F32) return append_t<float>(d, a, st);
  if (d->dtype == MA_ATTN_BF16) return append_t<__bf16>(d, a, st);
  return append_t<_Float16>(d, a, st);
}

size_t ma_paged_decode_workspace_size(const ma_paged_desc* d) {
  ma_host::clear_error();
  if (check(d, "ma_paged_decode_workspace_size")) return 0;
  const int64_t ns = decode_splits(d);
  if (ns <= 1) return 0;
  return (size_t)(d->batch * d->num_heads * ns) * (size_t)(d->head_dim + 2) * sizeof(float);
}

int ma_paged_decode(const ma_paged_desc* d, const void* query, const void* cache_key, const void* cache_value,
                    const int32_t* page_table, const int32_t* lengths, const int32_t* pages, void* out, float* lse,
                    void* workspace, size_t workspace_bytes, void* stream) {
  ma_host::clear_error();
  const char* who = "ma_paged_decode";
  if (check(d, who)) return 1;
  if (!(d->scale >= 0.0f) || std::isinf(d->scale)) return fail("%s: scale must be finite and >= 0", who);
  if (d->num_selected < 0 || d->num_selected > 64)
    return fail("%s: at most 64 listed pages, got %lld", who, (long long)d->num_selected);
  if ((pages != nullptr) != (d->num_selected > 0))
    return fail("%s: a page list and num_selected go together", who);
  if (pages && d->left >= 0) return fail("%s: listed pages take no window", who);
  if (d->num_global < 0 || (d->num_global > 0 && d->left < 0))
    return fail("%s: num_global must be >= 0 and goes with left >= 0", who);
  if (d->batch == 0) return 0;
  if (!query || !lengths || !out || (d->table_width && !page_table))
    return fail("%s: null pointer", who);
  if (d->num_pages < 1 || !cache_key || !cache_value) return fail("%s: the cache holds no page", who);
  for (const void* p : {query, cache_key, cache_value, (const void*)out})
    if (!aligned16(p)) return fail("%s: tensors must be 16-byte aligned", who);
  const int64_t ns = decode_splits(d);
  const size_t need = ma_paged_decode_workspace_size(d);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail("%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, need, workspace_bytes);
  DecodeArgs a{};
  a.q = query;
  a.ck = cache_key;
  a.cv = cache_value;
  a.table = page_table;
  a.lengths = lengths;
  a.pages = pages;
  a.out = out;
  a.lse = lse;
  a.num_pages = d->num_pages;
  a.width = (int32_t)d->table_width;
  a.page = (int32_t)d->page_size;
  a.H = (int32_t)d->num_heads;
  a.Hkv = (int32_t)d->num_kv_heads;
  a.G = a.H / a.Hkv;
  a.gt = (a.G + 15) / 16;
  a.D = (int32_t)d->head_dim;
  a.S = (int32_t)d->num_selected;
  a.nsplit = (int32_t)ns;
  a.windowed = d->left >= 0;
  a.left = d->left;
  a.nglobal = d->num_global;
  const float scale = d->scale > 0.0f ? d->scale : 1.0f / std::sqrt((float)a.D);
  a.scale_log2 = scale * 1.4426950408889634f;
  if (d->batch * a.Hkv * a.gt * ns > kMaxGrid || d->batch * a.H > kMaxGrid)
    return fail("%s: batch * heads too large", who);
  if (need) {
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)(d->batch * a.H * ns) * a.D;
  }
  Events ev(d);
  (void)hipGetLastError();
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->dtype == MA_ATTN_F32) return decode_t<float>(d, a, st);
  if (d->dtype == MA_ATTN_BF16) return decode_t<__bf16>(d, a, st);
  return decode_t<_Float16>(d, a, st);
}

int ma_paged_select(const ma_paged_desc* d, const void* query, const float* key_sums, const int32_t* page_table,
                    const int32_t* lengths, int32_t* pages, void* stream) {
  ma_host::clear_error();
  const char* who = "ma_paged_select";
  if (check(d, who)) return 1;
  if (d->num_selected < 1 || d->num_selected > 64)
    return fail("%s: num_selected must be in [1, 64], got %lld", who, (long long)d->num_selected);
  if (d->first_pages < 0 || d->local_pages < 1 || d->first_pages > 64 || d->local_pages > 64 ||
      d->first_pages + d->local_pages > d->num_selected)
    return fail("%s: first_pages >= 0 and local_pages >= 1 must fit in num_selected", who);
  if (d->table_width > 16384) return fail("%s: at most 16384 pages a stream, got %lld", who, (long long)d->table_width);
  if (d->batch == 0) return 0;
  if (!query || !key_sums || !lengths || !pages || (d->table_width && !page_table))
    return fail("%s: null pointer", who);
  if (!aligned16(key_sums) || !aligned16(query)) return fail("%s: tensors must be 16-byte aligned", who);
  SelectArgs a{};
  a.q = query;
  a.sums = key_sums;
  a.table = page_table;
  a.lengths = lengths;
  a.out = pages;
  a.num_pages = d->num_pages;
  a.width = (int32_t)d->table_width;
  a.page = (int32_t)d->page_size;
  a.H = (int32_t)d->num_heads;
  a.Hkv = (int32_t)d->num_kv_heads;
  a.G = a.H / a.Hkv;
  a.D = (int32_t)d->head_dim;
  a.S = (int32_t)d->num_selected;
  a.first = (int32_t)d->first_pages;
  a.local = (int32_t)d->local_pages;
  if (d->batch * a.Hkv > kMaxGrid) return fail("%s: batch * heads too large", who);
  Events ev(d);
  (void)hipGetLastError();
  hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t shm = (size_t)std::max<int64_t>(a.width, 1) * sizeof(uint64_t);
  const dim3 grid((unsigned)(d->batch * a.Hkv));
#define MA_SELECT(T, THREADS)                                                                                        \
  do {                                                                                                               \
    if (shm > 48 * 1024 && ma_host::reserve_lds(reinterpret_cast<const void*>(&page_select_kernel<T, THREADS>),      \
                                                16384 * sizeof(uint64_t), st))                                       \
      return 1;                                                                                                      \
    ma_host::launch(true, page_select_kernel<T, THREADS>, grid, dim3(THREADS), (uint32_t)shm, st, a);                \
  } while (0)
#define MA_SELECT_W(T)             \
  do {                             \
    if (d->table_width > kSelWide) \
      MA_SELECT(T, 1024);          \
    else                           \
      MA_SELECT(T, 512);           \
  } while (0)
  if (d->dtype == MA_ATTN_F32)
    MA_SELECT_W(float);
  else if (d->dtype == MA_ATTN_BF16)
    MA_SELECT_W(__bf16);
  else
    MA_SELECT_W(_Float16);
#undef MA_SELECT_W
#undef MA_SELECT
  return launched(who);
}

}  // extern "C"
