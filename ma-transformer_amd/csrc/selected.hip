// selected.hip -- ma_selected_forward / ma_selected_backward (ma_select.h):
// workspace layout and launches of selected_kernel.h.
#include "select_host.h"
#include "selected_kernel.h"

namespace {

using namespace ma_selected;
using namespace ma_select_host;

// The pairs' partial rows of the units that run together stay below this; a
// unit that is larger by itself runs alone.
constexpr size_t kPartBudget = (size_t)1 << 30;

struct Layout {
  Args a;
  int64_t units;
  int64_t group;  // units per launch
  size_t counts, offs, list, items, blk_items, part, ml, delta, part_kv, unread, total;
};

size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

// Pairs per item.  Enough items to fill the card several times over, but as
// few as possible beyond that: each reads its block again and, backward, leaves
// a part of dK and dV.
int pairs_per_item(const ma_select_desc* d, bool backward) {
  const int64_t G = d->num_heads / d->num_kv_heads;
  const int64_t rows = d->batch * d->num_heads * d->seq_len * d->num_selected;
  const int64_t most = backward ? 2048 : 512, least = backward ? 128 : 64;
  const int64_t want = std::min(most, std::max(least, rows / 2048));
  return (int)std::max<int64_t>(16, want / G);
}

Layout layout(const ma_select_desc* d, bool backward) {
  Layout l{};
  Args& a = l.a;
  a.N = d->seq_len;
  a.H = (int32_t)d->num_heads;
  a.Hkv = (int32_t)d->num_kv_heads;
  a.G = a.H / a.Hkv;
  a.D = (int32_t)d->head_dim;
  a.S = (int32_t)d->num_selected;
  a.BS = (int32_t)d->block_size;
  a.nb = (int32_t)blocks_of(d);
  a.causal = d->causal != 0;
  // chunks of 256 queries where their bitmap leaves room for two workgroups a CU
  a.words = a.nb <= 2048 ? 4 : 1;
  a.chunks = (int32_t)((a.N + 64 * a.words - 1) / (64 * a.words));
  a.cap = pairs_per_item(d, backward);
  a.max_items = (int32_t)(a.nb + a.N * a.S / a.cap);
  a.scale = d->scale > 0.0f ? d->scale : 1.0f / std::sqrt((float)a.D);
  a.scale_log2 = a.scale * 1.4426950408889634f;
  l.units = d->batch * a.Hkv;
  const size_t U = (size_t)l.units;
  const size_t pairs = (size_t)a.N * a.S * a.G;  // (pair, head) rows of a unit
  const size_t unit_part = pairs * a.D * sizeof(float);
  l.group = (int64_t)std::min<size_t>(U, std::max<size_t>(1, kPartBudget / std::max<size_t>(unit_part, 1)));
  const size_t g = (size_t)l.group;
  size_t o = 0;
  auto take = [&](size_t bytes) {
    const size_t at = o;
    o += up(bytes);
    return at;
  };
  l.counts = take(U * a.chunks * a.nb * sizeof(uint32_t));
  l.offs = take(U * a.nb * sizeof(int32_t));
  l.list = take(U * a.N * a.S * sizeof(int32_t));
  l.items = take(U * a.max_items * sizeof(int4));
  l.blk_items = take(U * a.nb * sizeof(int2));
  l.part = take(g * unit_part);
  if (backward) {
    l.delta = take((size_t)d->batch * a.N * a.H * sizeof(float));
    l.part_kv = take(g * a.max_items * 2 * a.BS * a.D * sizeof(float));
    l.unread = take(a.D * sizeof(float));
  } else {
    l.ml = take(g * pairs * sizeof(float2));
  }
  l.total = o;
  return l;
}

int place(Layout& l, const ma_select_desc* d, void* ws, size_t bytes, const char* who) {
  if (!ws || bytes < l.total || !aligned16(ws))
    return fail("%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, l.total, bytes);
  uint8_t* p = static_cast<uint8_t*>(ws);
  Args& a = l.a;
  a.counts = reinterpret_cast<uint32_t*>(p + l.counts);
  a.offs = reinterpret_cast<int32_t*>(p + l.offs);
  a.list = reinterpret_cast<int32_t*>(p + l.list);
  a.items = reinterpret_cast<int4*>(p + l.items);
  a.blk_items = reinterpret_cast<int2*>(p + l.blk_items);
  a.part = reinterpret_cast<float*>(p + l.part);
  a.ml = reinterpret_cast<float2*>(p + l.ml);
  a.delta = reinterpret_cast<float*>(p + l.delta);
  a.part_kv = reinterpret_cast<float*>(p + l.part_kv);
  a.unread = reinterpret_cast<float*>(p + l.unread);
  (void)d;
  return 0;
}

// Grids are 32-bit counts of workgroups of at most 1024 threads.
int check_grids(const Layout& l, const char* who) {
  const Args& a = l.a;
  const int64_t lim = INT32_MAX / 1024;
  if (l.units * a.chunks > lim || l.group * (int64_t)a.max_items > lim || l.group * (int64_t)a.nb * kKvParts > lim ||
      l.group * a.N * a.G / kJoinWaves > lim || (int64_t)a.N * a.S > INT32_MAX ||
      l.units / a.Hkv * a.N * a.H / 32 > lim)
    return fail("%s: batch * seq_len * heads too large", who);
  return 0;
}

int build_lists(const Layout& l, hipStream_t st) {
  const Args& a = l.a;
  const size_t bm = (size_t)a.nb * a.words * 8, tot = (size_t)a.nb * 4, fill = fill_lds_bytes(a.nb, a.words, a.S);
  static_assert(kMaxBlocks * 8 + 64 * 64 * 4 <= 160 * 1024 && 2048 * (4 * 8 + 4) + 256 * 64 * 4 <= 160 * 1024,
                "fill_kernel's LDS");
  if (bm > 48 * 1024 && ma_host::reserve_lds(reinterpret_cast<const void*>(&count_kernel), kMaxBlocks * 8, st))
    return 1;
  if (fill > 48 * 1024 &&
      ma_host::reserve_lds(reinterpret_cast<const void*>(&fill_kernel), kMaxBlocks * 8 + 64 * 64 * 4, st))
    return 1;
  if (tot > 48 * 1024 && ma_host::reserve_lds(reinterpret_cast<const void*>(&scan_kernel), kMaxBlocks * 4, st))
    return 1;
  const dim3 grid((unsigned)(l.units * a.chunks));
  ma_host::launch(false, count_kernel, grid, dim3(kListThreads), (uint32_t)bm, st, a);
  ma_host::launch(false, scan_kernel, dim3((unsigned)l.units), dim3(kScanThreads), (uint32_t)tot, st, a);
  ma_host::launch(false, fill_kernel, grid, dim3(kListThreads), (uint32_t)fill, st, a);
  return 0;
}

template <typename T, bool FWD>
void join(const Args& a, bool last, hipStream_t st) {
  const int64_t waves = (int64_t)a.units * a.N * a.G;
  const dim3 grid((unsigned)((waves + kJoinWaves - 1) / kJoinWaves)), block(64 * kJoinWaves);
  if (a.D <= 32)
    ma_host::launch(last, join_kernel<T, 8, FWD>, grid, block, 0, st, a);
  else if (a.D <= 64)
    ma_host::launch(last, join_kernel<T, 16, FWD>, grid, block, 0, st, a);
  else
    ma_host::launch(last, join_kernel<T, 32, FWD>, grid, block, 0, st, a);
}

template <typename T, int DP, int NT, bool FULL>
int forward_dn(Layout l, hipStream_t st) {
  Args a = l.a;
  for (int64_t u = 0; u < l.units; u += l.group) {
    a.unit0 = (int32_t)u;
    a.units = (int32_t)std::min(l.group, l.units - u);
    ma_host::launch(false, forward_kernel<T, DP, NT, FULL>, dim3((unsigned)(a.units * a.max_items)), dim3(64 * kFwdWaves), 0,
                    st, a);
    join<T, true>(a, u + l.group >= l.units, st);
  }
  return launched("ma_selected_forward");
}

template <typename T, int DP, int NT, bool FULL>
int backward_dn(Layout l, hipStream_t st) {
  Args a = l.a;
  constexpr size_t shm = BwdLds<T, DP, NT>::kBytes;
  if (shm > 48 * 1024 &&
      ma_host::reserve_lds(reinterpret_cast<const void*>(&backward_kernel<T, DP, NT, FULL>), shm, st))
    return 1;
  const int64_t rows = l.units / a.Hkv * a.N * a.H;
  ma_host::launch(false, delta_kernel<T>, dim3((unsigned)((rows * 8 + 255) / 256)), dim3(256), 0, st, a, rows);
  for (int64_t u = 0; u < l.units; u += l.group) {
    a.unit0 = (int32_t)u;
    a.units = (int32_t)std::min(l.group, l.units - u);
    ma_host::launch(false, backward_kernel<T, DP, NT, FULL>, dim3((unsigned)(a.units * a.max_items)), dim3(64 * NT),
                    (uint32_t)shm, st, a);
    ma_host::launch(false, join_kv_kernel<T>, dim3((unsigned)(a.units * a.nb * kKvParts)), dim3(256), 0, st, a);
    join<T, false>(a, u + l.group >= l.units, st);
  }
  return launched("ma_selected_backward");
}

template <typename T, int DP, bool BWD, bool FULL>
int run_df(const Layout& l, hipStream_t st) {
  if (l.a.BS == 16) return BWD ? backward_dn<T, DP, 1, FULL>(l, st) : forward_dn<T, DP, 1, FULL>(l, st);
  if (l.a.BS == 32) return BWD ? backward_dn<T, DP, 2, FULL>(l, st) : forward_dn<T, DP, 2, FULL>(l, st);
  return BWD ? backward_dn<T, DP, 4, FULL>(l, st) : forward_dn<T, DP, 4, FULL>(l, st);
}

// head_dim rounded up to DP; the kernels of exactly DP carry no tail.
template <typename T, int DP, bool BWD>
int run_d(const Layout& l, hipStream_t st) {
  return l.a.D == DP ? run_df<T, DP, BWD, true>(l, st) : run_df<T, DP, BWD, false>(l, st);
}

template <typename T, bool BWD>
int run_t(const Layout& l, hipStream_t st) {
  if (l.a.D <= 32) return run_d<T, 32, BWD>(l, st);
  if (l.a.D <= 64) return run_d<T, 64, BWD>(l, st);
  return run_d<T, 128, BWD>(l, st);
}

template <bool BWD>
int run(int dtype, const Layout& l, hipStream_t st) {
  if (build_lists(l, st)) return 1;
  if (dtype == MA_ATTN_F32) return run_t<float, BWD>(l, st);
  if (dtype == MA_ATTN_BF16) return run_t<__bf16, BWD>(l, st);
  return run_t<_Float16, BWD>(l, st);
}

int check_scale(const ma_select_desc* d, const char* who) {
  return !(d->scale >= 0.0f) || std::isinf(d->scale) ? fail("%s: scale must be finite and >= 0", who) : 0;
}

}  // namespace

extern "C" {

size_t ma_selected_forward_workspace_size(const ma_select_desc* d) {
  ma_host::clear_error();
  if (check(d, "ma_selected_forward_workspace_size") || !d->batch || !d->seq_len) return 0;
  return layout(d, false).total;
}

size_t ma_selected_backward_workspace_size(const ma_select_desc* d) {
  ma_host::clear_error();
  if (check(d, "ma_selected_backward_workspace_size") || !d->batch || !d->seq_len) return 0;
  return layout(d, true).total;
}

int ma_selected_forward(const ma_select_desc* d, const void* q, const void* k, const void* v, const int32_t* blocks,
                        void* o, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  ma_host::clear_error();
  const char* who = "ma_selected_forward";
  if (check(d, who) || check_scale(d, who)) return 1;
  if (!d->batch || !d->seq_len) return 0;
  if (check_aligned({q, k, v, o, blocks}, who)) return 1;
  Layout l = layout(d, false);
  if (check_grids(l, who) || place(l, d, workspace, workspace_bytes, who)) return 1;
  l.a.q = q;
  l.a.k = k;
  l.a.v = v;
  l.a.blocks = blocks;
  l.a.out = o;
  l.a.lse = lse;
  Events ev(d);
  (void)hipGetLastError();
  return run<false>(d->dtype, l, static_cast<hipStream_t>(stream));
}

int ma_selected_backward(const ma_select_desc* d, const void* q, const void* k, const void* v, const int32_t* blocks,
                         const void* o, const float* lse, const void* dout, void* dq, void* dk, void* dv,
                         void* workspace, size_t workspace_bytes, void* stream) {
  ma_host::clear_error();
  const char* who = "ma_selected_backward";
  if (check(d, who) || check_scale(d, who)) return 1;
  if (!d->batch || !d->seq_len) return 0;
  if (check_aligned({q, k, v, blocks, o, lse, dout, dq, dk, dv}, who)) return 1;
  Layout l = layout(d, true);
  if (check_grids(l, who) || place(l, d, workspace, workspace_bytes, who)) return 1;
  l.a.q = q;
  l.a.k = k;
  l.a.v = v;
  l.a.blocks = blocks;
  l.a.o = o;
  l.a.lse_in = lse;
  l.a.g = dout;
  l.a.dq = dq;
  l.a.dk = dk;
  l.a.dv = dv;
  Events ev(d);
  (void)hipGetLastError();
  return run<true>(d->dtype, l, static_cast<hipStream_t>(stream));
}

}  // extern "C"
