// select.hip -- ma_select_blocks (ma_select.h): launches of select_kernel.h.
#include "select_host.h"
#include "select_kernel.h"

namespace {

using namespace ma_select;
using namespace ma_select_host;

size_t mean_bytes(const ma_select_desc* d) {
  return (size_t)(d->batch * d->num_kv_heads * ((blocks_of(d) + 15) / 16 * 16) * d->head_dim) * sizeof(double);
}

template <typename T, int DP>
int rows_dp(const Args& a, int64_t grid, hipStream_t st) {
  const size_t shm = row_lds_bytes(a.S);
  if (shm > 48 * 1024 &&
      ma_host::reserve_lds(reinterpret_cast<const void*>(&rows_kernel<T, DP>), row_lds_bytes(64), st))
    return 1;
  ma_host::launch(true, rows_kernel<T, DP>, dim3((unsigned)grid), dim3(64 * kRowWaves), (uint32_t)shm, st, a);
  return 0;
}

template <typename T>
int select_t(const ma_select_desc* d, const Args& a, int64_t grid, hipStream_t st) {
  const int parts = (a.Hkv * a.D + kMeanThreads - 1) / kMeanThreads;
  ma_host::launch(false, mean_kernel<T>, dim3((unsigned)(d->batch * a.nbp * parts)), dim3(kMeanThreads), 0, st, a,
                  parts);
  const int rc = a.D <= 32   ? rows_dp<T, 32>(a, grid, st)
                 : a.D <= 64 ? rows_dp<T, 64>(a, grid, st)
                             : rows_dp<T, 128>(a, grid, st);
  return rc ? rc : launched("ma_select_blocks");
}

}  // namespace

extern "C" {

size_t ma_select_blocks_workspace_size(const ma_select_desc* d) {
  ma_host::clear_error();
  if (check(d, "ma_select_blocks_workspace_size")) return 0;
  return mean_bytes(d);
}

int ma_select_blocks(const ma_select_desc* d, const void* q, const void* k, int32_t* blocks, void* workspace,
                     size_t workspace_bytes, void* stream) {
  ma_host::clear_error();
  const char* who = "ma_select_blocks";
  if (check(d, who)) return 1;
  if (d->first_blocks < 0 || d->local_blocks < 1 || d->first_blocks > 64 || d->local_blocks > 64 ||
      d->first_blocks + d->local_blocks > d->num_selected)
    return fail("%s: first_blocks >= 0 and local_blocks >= 1 must fit in num_selected", who);
  if (d->batch == 0 || d->seq_len == 0) return 0;
  if (check_aligned({q, k, blocks}, who)) return 1;
  if (!workspace || workspace_bytes < mean_bytes(d) || !aligned16(workspace))
    return fail("%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, mean_bytes(d), workspace_bytes);
  Args a{};
  a.q = q;
  a.k = k;
  a.mean = static_cast<double*>(workspace);
  a.out = blocks;
  a.N = d->seq_len;
  a.units = (int32_t)std::min<int64_t>(d->batch * d->num_kv_heads, INT32_MAX);
  a.H = (int32_t)d->num_heads;
  a.Hkv = (int32_t)d->num_kv_heads;
  a.G = a.H / a.Hkv;
  a.D = (int32_t)d->head_dim;
  a.S = (int32_t)d->num_selected;
  a.BS = (int32_t)d->block_size;
  a.nb = (int32_t)blocks_of(d);
  a.nbp = (a.nb + 15) / 16 * 16;
  a.causal = d->causal != 0;
  a.first = (int32_t)d->first_blocks;
  a.local = (int32_t)d->local_blocks;
  const int64_t waves = d->batch * d->num_kv_heads * ((d->seq_len + 15) / 16);
  const int64_t grid = (waves + kRowWaves - 1) / kRowWaves;
  const int64_t mean_grid = d->batch * a.nbp * ((a.Hkv * a.D + kMeanThreads - 1) / kMeanThreads);
  if (grid > INT32_MAX / 256 || mean_grid > INT32_MAX / 256) return fail("%s: batch * seq_len * heads too large", who);
  Events ev(d);
  (void)hipGetLastError();
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (d->dtype == MA_ATTN_F32) return select_t<float>(d, a, grid, st);
  if (d->dtype == MA_ATTN_BF16) return select_t<__bf16>(d, a, grid, st);
  return select_t<_Float16>(d, a, grid, st);
}

}  // extern "C"
