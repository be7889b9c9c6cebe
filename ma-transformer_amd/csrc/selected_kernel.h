// selected_kernel.h -- attention of each query over its own listed blocks.
//
// Both directions run key block by key block: the (query, slot) pairs that
// list a block are gathered into a list, so that a block's keys and values are
// read once per a few hundred queries and the products are dense MFMA tiles.
// Going query by query instead would read block_size keys and values per pair
// (16 KB at 64 x 64 in 16 bits) where this reads a query row and writes one
// float32 partial row.  What a pair produces for its query (forward: maximum,
// sum and output of its block; backward: its part of dQ) goes to the pair's
// own place in the workspace, and a second kernel joins the slots of a query
// in slot order: no atomics, the same bits every time.
//
// A unit is one (batch, key/value head).  Lists are ascending in the query, so
// the sums over a list have a fixed order too.
#pragma once

#include "attn_planes.h"
#include "device_common.h"

namespace ma_selected {

using namespace ma_dev;

struct Args {
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* g;  // output gradient
  const int32_t* blocks;
  void* out;   // forward: o
  void* dq;
  void* dk;
  void* dv;
  const float* lse_in;
  float* lse;
  // index: per unit
  uint32_t* counts;  // [chunks][nb] pairs of the chunk's queries per block, then their prefix
  int32_t* offs;     // [nb] where a block's list begins
  int32_t* list;     // [N * S] query * 64 + slot
  int4* items;       // [max_items] {block, first pair, pairs, place among the block's items}; pairs < 0: none
  int2* blk_items;   // [nb] {first item, items}
  float* part;       // group's pairs: [N][S][G][D]
  float2* ml;        // [N][S][G]
  float* delta;      // [B][N][H]
  float* part_kv;    // group's items: [max_items][2][BS][D]
  float* unread;     // [D] written and never read
  int64_t N;
  int32_t H, Hkv, G, D, S, BS, nb, causal;
  int32_t chunks, words, max_items, cap;  // cap: pairs per item
  int32_t unit0, units;                   // units of this launch
  float scale, scale_log2;
};

// ---------------------------------------------------------------- lists
//
// A chunk of 64 * words queries marks its pairs in an LDS bitmap (a bit per
// query and block: setting bits commutes, and repeats fall together); counts
// and ranks are population counts, so the lists come out in query order
// whatever order the threads run in.  8 heads of 16384 queries, 16 of 256 blocks:
// 7 + 8 + 22 us.

constexpr int kListThreads = 1024;
constexpr int kScanThreads = 1024;

// Entry j of a query's list: its block, or -1 where it is skipped.
__device__ __forceinline__ int listed(const Args& a, const int32_t* row, int64_t i, int j) {
  const int32_t b = row[j];
  if (b < 0 || b >= a.nb || (a.causal && (int64_t)b * a.BS > i)) return -1;
  return b;
}

__device__ __forceinline__ const int32_t* row_of(const Args& a, int unit, int64_t i) {
  return a.blocks + (((int64_t)(unit / a.Hkv) * a.N + i) * a.Hkv + unit % a.Hkv) * a.S;
}

__global__ __launch_bounds__(kListThreads) void count_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  unsigned long long* bm = reinterpret_cast<unsigned long long*>(lds);
  const uint32_t x = (uint32_t)xcd_row_order((int)blockIdx.x, (int)gridDim.x);
  const int unit = x / (uint32_t)a.chunks, ch = x % (uint32_t)a.chunks;
  const int64_t q0 = (int64_t)ch * 64 * a.words;
  const int nq = (int)(a.N - q0 < 64 * a.words ? a.N - q0 : 64 * a.words);
  for (int i = threadIdx.x; i < a.nb * a.words; i += kListThreads) bm[i] = 0;
  __syncthreads();
  for (int e = threadIdx.x; e < nq * a.S; e += kListThreads) {
    const int qi = e / a.S, j = e - qi * a.S;
    const int b = listed(a, row_of(a, unit, q0 + qi), q0 + qi, j);
    if (b >= 0) atomicOr(&bm[b * a.words + (qi >> 6)], 1ull << (qi & 63));
  }
  __syncthreads();
  uint32_t* out = a.counts + ((int64_t)unit * a.chunks + ch) * a.nb;
  for (int b = threadIdx.x; b < a.nb; b += kListThreads) {
    uint32_t n = 0;
    for (int w = 0; w < a.words; ++w) n += (uint32_t)__popcll(bm[b * a.words + w]);
    out[b] = n;
  }
}

// Per unit: each block's chunk counts to prefixes, list offsets, work items.
__global__ __launch_bounds__(kScanThreads) void scan_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  uint32_t* tot = reinterpret_cast<uint32_t*>(lds);  // [nb]
  __shared__ uint32_t s_wave[2][kScanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, unit = blockIdx.x;
  uint32_t* cnt = a.counts + (int64_t)unit * a.chunks * a.nb;
  for (int b = tid; b < a.nb; b += kScanThreads) {
    uint32_t run = 0;
    for (int c0 = 0; c0 < a.chunks; c0 += 16) {  // sixteen loads in flight
      uint32_t x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = c0 + i < a.chunks ? cnt[(int64_t)(c0 + i) * a.nb + b] : 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (c0 + i < a.chunks) cnt[(int64_t)(c0 + i) * a.nb + b] = run;
        run += x[i];
      }
    }
    tot[b] = run;
  }
  __syncthreads();
  // each thread's run of consecutive blocks, then a scan over the threads
  const int per = (a.nb + kScanThreads - 1) / kScanThreads;
  const int b0 = tid * per < a.nb ? tid * per : a.nb, b1 = b0 + per < a.nb ? b0 + per : a.nb;
  uint32_t pairs = 0, items = 0;
  for (int b = b0; b < b1; ++b) {
    pairs += tot[b];
    items += tot[b] ? (tot[b] + a.cap - 1) / a.cap : 1;  // an empty list is an item: its dK, dV are zeros
  }
  uint32_t x[2] = {pairs, items};
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const uint32_t own = x[y];
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const uint32_t z = __shfl_up(x[y], k, 64);
      if (lane >= k) x[y] += z;
    }
    if (lane == 63) s_wave[y][tid >> 6] = x[y];
    x[y] -= own;
  }
  __syncthreads();
  uint32_t total = 0;
  for (int w = 0; w < kScanThreads / 64; ++w) {
    if (w < (tid >> 6)) x[0] += s_wave[0][w], x[1] += s_wave[1][w];
    total += s_wave[1][w];
  }
  int4* it = a.items + (int64_t)unit * a.max_items;
  for (int b = b0; b < b1; ++b) {
    a.offs[(int64_t)unit * a.nb + b] = (int32_t)x[0];
    const int n = tot[b] ? (int)((tot[b] + a.cap - 1) / a.cap) : 1;
    a.blk_items[(int64_t)unit * a.nb + b] = make_int2((int)x[1], n);
    for (int i = 0; i < n; ++i) {
      const int left = (int)tot[b] - i * a.cap;
      it[x[1] + i] = make_int4(b, (int)x[0] + i * a.cap, left < a.cap ? left : a.cap, i);
    }
    x[0] += tot[b];
    x[1] += n;
  }
  for (int i = (int)total + tid; i < a.max_items; i += kScanThreads) it[i] = make_int4(0, 0, -1, 0);
}

// dynamic LDS of fill_kernel: the bitmap, the chunk's rows, and (small tables)
// where each block's pairs of this chunk begin
inline size_t fill_lds_bytes(int nb, int words, int S) {
  return (size_t)nb * words * 8 + (size_t)64 * words * S * 4 + (words > 1 ? (size_t)nb * 4 : 0);
}

__global__ __launch_bounds__(kListThreads) void fill_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  unsigned long long* bm = reinterpret_cast<unsigned long long*>(lds);
  int32_t* rows = reinterpret_cast<int32_t*>(bm + a.nb * a.words);
  uint32_t* begin = reinterpret_cast<uint32_t*>(rows + 64 * a.words * a.S);
  const uint32_t x = (uint32_t)xcd_row_order((int)blockIdx.x, (int)gridDim.x);
  const int unit = x / (uint32_t)a.chunks, ch = x % (uint32_t)a.chunks;
  const int64_t q0 = (int64_t)ch * 64 * a.words;
  const int nq = (int)(a.N - q0 < 64 * a.words ? a.N - q0 : 64 * a.words);
  const uint32_t* base = a.counts + ((int64_t)unit * a.chunks + ch) * a.nb;
  const int32_t* offs = a.offs + (int64_t)unit * a.nb;
  const bool staged = a.words > 1;
  if (staged)
    for (int i = threadIdx.x; i < a.nb; i += kListThreads) begin[i] = base[i] + (uint32_t)offs[i];
  for (int i = threadIdx.x; i < a.nb * a.words; i += kListThreads) bm[i] = 0;
  __syncthreads();
  for (int e = threadIdx.x; e < nq * a.S; e += kListThreads) {
    const int qi = e / a.S, j = e - qi * a.S;
    const int b = listed(a, row_of(a, unit, q0 + qi), q0 + qi, j);
    rows[e] = b;
    if (b >= 0) atomicOr(&bm[b * a.words + (qi >> 6)], 1ull << (qi & 63));
  }
  __syncthreads();
  int32_t* list = a.list + (int64_t)unit * a.N * a.S;
  for (int e = threadIdx.x; e < nq * a.S; e += kListThreads) {
    const int b = rows[e];
    if (b < 0) continue;
    const int qi = e / a.S, j = e - qi * a.S;
    bool again = false;  // an earlier entry of the row is this block
    for (int i = 0; i < j; ++i) again = again || rows[e - j + i] == b;
    if (again) continue;
    uint32_t rank = staged ? begin[b] : base[b] + (uint32_t)offs[b];
    for (int w = 0; w < (qi >> 6); ++w) rank += (uint32_t)__popcll(bm[b * a.words + w]);
    rank += (uint32_t)__popcll(bm[b * a.words + (qi >> 6)] & ((1ull << (qi & 63)) - 1));
    list[rank] = (int32_t)((q0 + qi) * 64 + j);
  }
}

// ---------------------------------------------------------------- forward
//
// One workgroup takes an item: up to `cap` pairs of one block.  Each wave keeps
// the block's keys and values as MFMA operands in registers and goes through
// tiles of 16 (pair, head) rows: S^T = K Q^T has a row in each column and
// four keys of each 16-key tile in each lane, the operand layout of
// O^T = V^T P^T, so statistics and weights never leave their lane.
//
// Bound by the partial rows (one float32 row of head_dim per pair and head,
// written here and read by the join): without its stores the kernel takes 107
// us where it takes 135 to 150 (8 heads of 16384 rows, 16 of 64 keys, bf16: 537
// MB of partial rows, 4.0 TB/s).  They go through LDS so that a store writes
// whole rows, and past the caches (non-temporal): half rows stored from the
// result layout took 230 us, whole rows 205, and the join reads them in 125
// instead of 145.

constexpr int kFwdWaves = 4;

// Value rows 4 g + i of a 16-key tile as the words the lane loads, and the V^T
// operands built from two such tiles.  Lane column c takes the 4 (VPL = 2: 2)
// elements at 4 p(c), p(c) = 4 (c % 4) + c / 4, of each 64 (32): a result's rows
// 4 g + y are then elements at 4 (4 y + g), and the four lanes that share a row
// store 64 contiguous bytes at once.
template <typename T, int DP>
struct ValueRows {
  static constexpr int VPL = DP / 16;
  static constexpr int VW = VPL * (int)sizeof(T) / 4;
  uint32_t w[4][VW];
  static constexpr int CH = VPL < 4 ? VPL : 4;        // elements of a chunk
  static constexpr int CW = CH * (int)sizeof(T) / 4;  // words of it
  __device__ __forceinline__ void load(int i, const T* row, bool ok, int c, int D) {
#pragma unroll
    for (int h = 0; h < VPL / CH; ++h) {
      const int d = 16 * CH * h + CH * (4 * (c & 3) + (c >> 2));
      const uint32_t* p = reinterpret_cast<const uint32_t*>(row + (d < D ? d : 0));
      const bool in = ok && d < D;
      if constexpr (CW == 1) {
        w[i][h] = p[0];
      } else if constexpr (CW == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[i][2 * h] = x.x, w[i][2 * h + 1] = x.y;
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[i][4 * h] = x.x, w[i][4 * h + 1] = x.y, w[i][4 * h + 2] = x.z, w[i][4 * h + 3] = x.w;
      }
#pragma unroll
      for (int y = 0; y < CW; ++y) w[i][CW * h + y] = in ? w[i][CW * h + y] : 0u;
    }
  }
  // the head_dim element of result row 4 g + y of operand j
  static __device__ __forceinline__ int element(int g, int y, int j) {
    return 16 * CH * (j / CH) + CH * (4 * y + g) + j % CH;
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int y = 0; y < VW; ++y) w[i][y] = 0;
  }
};

// Operand j from the tiles u0 and u1.
template <typename T, int DP>
__device__ __forceinline__ typename Op<T>::F value_operand(const ValueRows<T, DP>& u0, const ValueRows<T, DP>& u1, int j) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
    return make_uint4(__builtin_amdgcn_perm(u0.w[1][j / 2], u0.w[0][j / 2], sel),
                      __builtin_amdgcn_perm(u0.w[3][j / 2], u0.w[2][j / 2], sel),
                      __builtin_amdgcn_perm(u1.w[1][j / 2], u1.w[0][j / 2], sel),
                      __builtin_amdgcn_perm(u1.w[3][j / 2], u1.w[2][j / 2], sel));
  } else {
    F32x8 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = __uint_as_float(u0.w[i][j]), f.v[4 + i] = __uint_as_float(u1.w[i][j]);
    return f;
  }
}

__device__ __forceinline__ int wave_any(bool x) { return __ballot(x) != 0; }

// Waves per SIMD that the registers are budgeted for; two or more keep the
// products out of the accumulation registers, whose copies cost as much as the
// products themselves.
template <typename T, int DP, int NT>
constexpr int kFwdOcc = DP * NT * (int)sizeof(T) > 512 ? (DP * NT * (int)sizeof(T) > 1024 ? 1 : 2) : 3;
template <typename T, int DP, int NT>
constexpr int kBwdRows = 32;  // rows of a backward tile
template <typename T, int DP, int NT>
constexpr int kBwdOcc = DP > 64 || (sizeof(T) == 4 && DP == 64 && NT == 1) ? 1 : (sizeof(T) == 2 && NT > 1 ? 3 : 2);

template <typename T, int DP, int NT, bool FULL>
__global__ __launch_bounds__(64 * kFwdWaves, (kFwdOcc<T, DP, NT>)) void forward_kernel(Args a) {
  using O = Op<T>;
  using F = typename O::F;
  using W = WeightPlanes<T>;
  using VR = ValueRows<T, DP>;
  constexpr int NK = DP / 32, NP = (NT + 1) / 2, VPL = VR::VPL;
  __shared__ __attribute__((aligned(16))) float tile_o[kFwdWaves][16][DP + 4];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int x = (int)blockIdx.x;
  const int ug = x / a.max_items, unit = a.unit0 + ug;
  const int4 item = a.items[(int64_t)unit * a.max_items + x % a.max_items];
  const int rows = item.z * a.G;
  if (rows <= 16 * w) return;
  const int b = unit / a.Hkv, hk = unit % a.Hkv, D = FULL ? DP : a.D, blk = item.x;
  const int64_t k0 = (int64_t)blk * a.BS, rs = (int64_t)a.Hkv * D;
  const T* kp = static_cast<const T*>(a.k) + (int64_t)b * a.N * rs + hk * D;
  const T* vp = static_cast<const T*>(a.v) + (int64_t)b * a.N * rs + hk * D;
  const int nk = (int)(a.N - k0 < 16 * NT ? a.N - k0 : 16 * NT);  // keys of the block

  F kf[NT][NK], vf[NP][VPL];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int key = 16 * t + c < nk ? 16 * t + c : nk - 1;
#pragma unroll
    for (int i = 0; i < NK; ++i)
      kf[t][i] = 32 * i + 8 * g < D ? O::load(kp + (k0 + key) * rs + 32 * i + 8 * g) : O::zero();
  }
  int vbad = 0;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    VR u[2];
    u[1].zero();
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (2 * p + h < NT) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = 16 * (2 * p + h) + 4 * g + i;
          u[h].load(i, vp + (k0 + (key < nk ? key : nk - 1)) * rs, key < nk, c, D);
        }
      }
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      vf[p][j] = value_operand<T, DP>(u[0], u[1], j);
      if (a.causal) vbad |= O::bad(vf[p][j]);
    }
  }
  vbad = wave_any(vbad);

  const int32_t* list = a.list + (int64_t)unit * a.N * a.S + item.y;
  // rows are addressed as 32-bit row numbers times 32-bit row bytes
  const uint8_t* qp = static_cast<const uint8_t*>(a.q) + ((int64_t)b * a.N * a.H + (int64_t)hk * a.G) * D * sizeof(T);
  const uint32_t qbytes = (uint32_t)(a.H * D) * sizeof(T), pbytes = (uint32_t)(a.G * D) * 4;
  uint8_t* part = reinterpret_cast<uint8_t*>(a.part + (int64_t)ug * a.N * a.S * a.G * D);
  float2* ml = a.ml + (int64_t)ug * a.N * a.S * a.G;
  const float sl2 = a.scale_log2;

  // a row past the end repeats the last one and stores the same values to the
  // same place, so that no store stands under a branch
  auto entry_of = [&](int r) { return list[(a.G == 1 ? r : r / a.G)]; };
  auto head_of = [&](int r) { return a.G == 1 ? 0 : r % a.G; };
  auto clamp = [&](int r) { return r < rows ? r : rows - 1; };
  // a tile's pairs are read two tiles ahead, its queries one
  constexpr int STEP = 16 * kFwdWaves;
  F qf[NK];
  int ent = entry_of(clamp(16 * w + c)), gh = head_of(clamp(16 * w + c));
  int entn = entry_of(clamp(16 * w + c + STEP));
  auto load_q = [&](F(&f)[NK], int e, int h) {
    const T* p = reinterpret_cast<const T*>(qp + (uint64_t)(uint32_t)(e >> 6) * qbytes + (uint32_t)(h * D) * sizeof(T));
#pragma unroll
    for (int i = 0; i < NK; ++i) f[i] = FULL || 32 * i + 8 * g < D ? O::load(p + 32 * i + 8 * g) : O::zero();
  };
  load_q(qf, ent, gh);
  for (int t0 = 16 * w; t0 < rows; t0 += STEP) {
    const int ghn = head_of(clamp(t0 + STEP + c));
    const int ent2 = entry_of(clamp(t0 + 2 * STEP + c));
    f32x4 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NK; ++i) s[t] = O::mma(kf[t][i], qf[i], s[t]);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) settle(s[t]);
    load_q(qf, entn, ghn);
    // keys of this row: up to its own (causal), up to the block's end
    const int qi = ent >> 6;
    int lim = nk;
    if (a.causal && qi - (int)k0 + 1 < lim) lim = qi - (int)k0 + 1;
    const bool masked = wave_any(lim < 16 * NT);
    if (masked) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[t][y] = 16 * t + 4 * g + y < lim ? s[t][y] : -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int y = 0; y < 4; ++y) m = fmaxf(m, s[t][y]);
    m = col_max(m) * sl2;  // the scale is positive
    const float mu = m == -INFINITY ? 0.0f : m - W::kBias;
    float p[2 * NP][4], l = 0.0f;
#pragma unroll
    for (int t = 0; t < 2 * NP; ++t)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        p[t][y] = t < NT ? __builtin_amdgcn_exp2f(fmaf(s[t < NT ? t : 0][y], sl2, -mu)) : 0.0f;
        l += p[t][y];
      }
    l = col_sum(l);
    f32x4 acc[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) acc[j] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      W pp;
      pp.set(p[2 * u], p[2 * u + 1]);
#pragma unroll
      for (int j = 0; j < VPL; ++j)
#pragma unroll
        for (int pl = W::N - 1; pl >= 0; --pl) acc[j] = O::mma(vf[u][j], pp.w[pl], acc[j]);
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) settle(acc[j]);
    if (__builtin_expect(masked && vbad, 0)) {
      // an infinite or NaN value behind a row's last key must not reach it:
      // weight by weight, allowed keys only
#pragma unroll
      for (int j = 0; j < VPL; ++j) acc[j] = f32x4{0, 0, 0, 0};
      for (int key = 0; key < nk; ++key) {
        float pk = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int y = 0; y < 4; ++y)
            if (t == key >> 4 && y == (key & 3)) pk = p[t][y];
        pk = __shfl(pk, c + 16 * ((key & 15) >> 2), 64);
        const T* row = vp + (k0 + key) * rs;
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int j = 0; j < VPL; ++j) {
            const int d = VR::element(g, y, j);
            if (key < lim && d < D) acc[j][y] += pk * (float)row[d];
          }
      }
    }
    // through LDS, so that a store writes whole rows
    const uint32_t pair = __umul24(qi, a.S) + (ent & 63);
    float* mine = &tile_o[w][c][0];
#pragma unroll
    for (int y = 0; y < 4; ++y)
#pragma unroll
      for (int j = 0; j < VPL; j += VR::CH) {
        const int d = VR::element(g, y, j);
        if constexpr (VPL == 2)
          *reinterpret_cast<float2*>(mine + d) = make_float2(acc[0][y], acc[1][y]);
        else
          *reinterpret_cast<float4*>(mine + d) = make_float4(acc[j][y], acc[j + 1][y], acc[j + 2][y], acc[j + 3][y]);
      }
    ml[(int64_t)pair * a.G + gh] = make_float2(m, l);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    constexpr int CPR = DP / 4, RPI = 64 / CPR;  // 16-byte chunks of a row, rows of a store
#pragma unroll
    for (int it = 0; it < 16 / RPI; ++it) {
      const int row = it * RPI + lane / CPR, d = (lane % CPR) * 4;
      const uint32_t pr = __shfl((int)pair, row, 64);
      const int gr = a.G == 1 ? 0 : __shfl(gh, row, 64);
      float* po = reinterpret_cast<float*>(part + (uint64_t)pr * pbytes) + gr * D + d;
      if (FULL || d < D)
        __builtin_nontemporal_store(*reinterpret_cast<const f32x4*>(&tile_o[w][row][d]), reinterpret_cast<f32x4*>(po));
    }
    __builtin_amdgcn_wave_barrier();
    ent = entn;
    entn = ent2;
    gh = ghn;
  }
}

// ---------------------------------------------------------------- joining a query's slots
//
// One wave per (unit, query, head).  Forward: o = sum 2^(m_s - M) o_s / sum
// 2^(m_s - M) l_s over the listed slots; backward: dQ = sum of the slots'
// parts.  Lanes hold four elements each; 64 / LP slots at once, four such rounds
// of loads ahead of their weights, past the caches (the rows are read once).
// 537 MB of partial rows: 125 us forward (4.3 TB/s), 96 backward (5.6).

constexpr int kJoinWaves = 4;

template <typename T, int LP, bool FWD>
__global__ __launch_bounds__(64 * kJoinWaves) void join_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t per = a.N * a.G;
  const int64_t id = (int64_t)blockIdx.x * kJoinWaves + (threadIdx.x >> 6);
  if (id >= per * a.units) return;
  const int ug = (int)(id / per), unit = a.unit0 + ug;
  const int64_t rem = id - ug * per, i = rem / a.G;
  const int gh = (int)(rem - i * a.G), D = a.D;
  const int b = unit / a.Hkv, hk = unit % a.Hkv;
  const int32_t* row = row_of(a, unit, i);
  const int64_t at = (((int64_t)ug * a.N + i) * a.S) * a.G + gh;  // slot s at + s * G
  float2 x = make_float2(-INFINITY, 0.0f);
  if (FWD && lane < a.S) x = a.ml[at + (int64_t)lane * a.G];  // not yet known to be written
  int e = lane < a.S ? listed(a, row, i, lane) : -1;
  for (int j = 0; j + 1 < a.S; ++j) {
    const int o = __builtin_amdgcn_readlane(e, j);
    if (j < lane && o == e) e = -1;
  }
  const uint64_t live = __ballot(e >= 0);
  // sixteen loads' worth of slots before their weights are needed
  constexpr int SL = 64 / LP;  // slots at once
  const int d = 4 * (lane & (LP - 1));
  const float* po = a.part + at * D + d;
  const int64_t sstep = (int64_t)a.G * D;
  float f = 1.0f, M = 0.0f, lt = 0.0f;
  float4 acc = make_float4(0, 0, 0, 0);
  for (int s0 = 0; s0 < a.S; s0 += 4 * SL) {
    f32x4 v[4];
    bool in[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int s = s0 + y * SL + lane / LP;
      in[y] = s < a.S && (live >> s & 1) && d < D;
      v[y] = f32x4{0, 0, 0, 0};
      if (in[y]) v[y] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(po + s * sstep));
    }
    if (FWD && s0 == 0) {
      if (e < 0) x = make_float2(-INFINITY, 0.0f);
      M = x.x;
#pragma unroll
      for (int k = 32; k >= 1; k >>= 1) M = fmaxf(M, __shfl_xor(M, k, 64));
      const float mu = M == -INFINITY ? 0.0f : M;
      f = e >= 0 ? __builtin_amdgcn_exp2f(x.x - mu) : 0.0f;
      lt = e >= 0 ? f * x.y : 0.0f;
#pragma unroll
      for (int k = 32; k >= 1; k >>= 1) lt += __shfl_xor(lt, k, 64);
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const float fs = FWD ? __shfl(f, (s0 + y * SL + lane / LP) & 63, 64) : 1.0f;
      if (in[y]) {
        acc.x += fs * v[y][0];
        acc.y += fs * v[y][1];
        acc.z += fs * v[y][2];
        acc.w += fs * v[y][3];
      }
    }
  }
#pragma unroll
  for (int k = LP; k < 64; k <<= 1) {
    acc.x += __shfl_xor(acc.x, k, 64);
    acc.y += __shfl_xor(acc.y, k, 64);
    acc.z += __shfl_xor(acc.z, k, 64);
    acc.w += __shfl_xor(acc.w, k, 64);
  }
  const int64_t orow = ((int64_t)b * a.N + i) * a.H + (int64_t)hk * a.G + gh;
  if (lane < LP && d < D) {
    T r[4];
    const float inv = FWD ? (live ? 1.0f / lt : 0.0f) : a.scale;
    if (FWD && !live) acc = make_float4(0, 0, 0, 0);
    r[0] = static_cast<T>(acc.x * inv);
    r[1] = static_cast<T>(acc.y * inv);
    r[2] = static_cast<T>(acc.z * inv);
    r[3] = static_cast<T>(acc.w * inv);
    T* op = static_cast<T*>(FWD ? a.out : a.dq) + orow * D + d;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(op) = *reinterpret_cast<const uint2*>(r);
    else
      *reinterpret_cast<uint4*>(op) = *reinterpret_cast<const uint4*>(r);
  }
  if (FWD && a.lse && lane == 0)
    a.lse[orow] = live ? M + (__log2f(lt) - WeightPlanes<T>::kBias) : -INFINITY;
}

// ---------------------------------------------------------------- backward

// delta = dO . O of every (batch, query, head), eight lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void delta_kernel(Args a, int64_t rows) {
  const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 3;
  const int e = threadIdx.x & 7;
  if (r >= rows) return;
  const T* o = static_cast<const T*>(a.o) + r * a.D;
  const T* g = static_cast<const T*>(a.g) + r * a.D;
  float s = 0.0f;
  for (int d = 8 * e; d < a.D; d += 64) {
    T x[8], y[8];
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(o + d);
      *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(g + d);
    } else {
      reinterpret_cast<uint4*>(x)[0] = reinterpret_cast<const uint4*>(o + d)[0];
      reinterpret_cast<uint4*>(x)[1] = reinterpret_cast<const uint4*>(o + d)[1];
      reinterpret_cast<uint4*>(y)[0] = reinterpret_cast<const uint4*>(g + d)[0];
      reinterpret_cast<uint4*>(y)[1] = reinterpret_cast<const uint4*>(g + d)[1];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s += (float)x[j] * (float)y[j];
  }
#pragma unroll
  for (int k = 1; k < 8; k <<= 1) s += __shfl_xor(s, k, 64);
  if (e == 0) a.delta[r] = s;
}

// f16's dS take a power of two: its largest magnitude so far in [2^13, 2^14),
// see backward_kernel.
template <typename T>
constexpr bool kScaled = __is_same(T, _Float16);

// One workgroup per item, wave w on the block's keys 16 w .. 16 w + 15, tiles of
// 32 (pair, head) rows whose Q and dO go through LDS.  With A = rows and
// B = keys, S and dP have a key in each column and four rows of each 16-row
// tile in each lane: the operand layout of dV^T = dO^T P and dK^T = Q^T dS,
// whose other operand is the transposed LDS read of the same tiles.  dS goes
// once through LDS for dQ^T = K^T dS^T, where wave w takes the head_dim tiles w,
// w + NT, ...  P and dS enter as planes (attn_planes.h).
//
// 8 heads of 16384 queries, 16 of 64 keys, bf16: 373 us.  Vector instructions
// take 47 % of its cycles, LDS 51 %, the matrix cores 27 %; dQ's partial rows
// (537 MB) would take 110 us at 5 TB/s.
//
// f16 has no bits below 2^-24, so its dS carry a power of two, common to the
// workgroup and only ever lowered: dK's sums are rescaled when a larger dS
// arrives, a tile's dQ is scaled back as it is stored.  A row keeps eleven bits
// (f16's own) down to 2^-27 of the item's largest dS.
template <typename T, int DP, int NT>
struct BwdLds {
  static constexpr int RT = kBwdRows<T, DP, NT>;
  static constexpr int RS = DP * (int)sizeof(T) + 16;       // bytes of a staged row
  static constexpr int SS = RT * (int)sizeof(T) + 16;       // bytes of a key's dS
  static constexpr int kQ = 0;
  static constexpr int kG = RT * RS;
  static constexpr int kS = 2 * RT * RS;
  static constexpr int kSPlane = 16 * NT * SS;
  static constexpr int kStat = kS + WeightPlanes<T>::N * kSPlane;  // lse, delta, pair, last key [RT]
  static constexpr int kMax = kStat + 4 * RT * 4;                  // [NT] per-wave maxima
  static constexpr int kFlag = kMax + NT * 4;                      // [2] tile flags, block flag
  static constexpr int kBytes = kFlag + 16;
};

template <typename T, int DP, int NT, bool FULL>
__global__ __launch_bounds__(64 * NT, (kBwdOcc<T, DP, NT>)) void backward_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  using O = Op<T>;
  using F = typename O::F;
  using W = WeightPlanes<T>;
  using L = BwdLds<T, DP, NT>;
  constexpr int NK = DP / 32, ND = DP / 16, RT = L::RT;
  constexpr int TH = 64 * NT, CPR = DP / 8, NC = (RT * CPR + TH - 1) / TH;  // staged chunks per thread
  constexpr int JD = (ND + NT - 1) / NT, KC = (NT + 1) / 2;
  static_assert(RT <= TH && RT % 32 == 0, "a thread per row of the tile");
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, c = lane & 15, g = lane >> 4;
  // whole units per XCD, whose L2 then holds their Q and dO (8 units of 16384
  // rows: training step 820 -> 790 us; 8 of 4095: 421 -> 424).  Other counts
  // would give one XCD a unit's first blocks, which have the longest lists.
  const int x = a.units % 8 == 0 ? xcd_row_order((int)blockIdx.x, (int)gridDim.x) : (int)blockIdx.x;
  const int ug = x / a.max_items, unit = a.unit0 + ug, slot_item = x % a.max_items;
  const int4 item = a.items[(int64_t)unit * a.max_items + slot_item];
  if (item.z < 0) return;
  const int rows = item.z * a.G;
  const int b = unit / a.Hkv, hk = unit % a.Hkv, D = FULL ? DP : a.D, blk = item.x;
  const int k0 = blk * a.BS;
  const int64_t rs = (int64_t)a.Hkv * D;
  const T* kp = static_cast<const T*>(a.k) + ((int64_t)b * a.N + k0) * rs + hk * D;
  const T* vp = static_cast<const T*>(a.v) + ((int64_t)b * a.N + k0) * rs + hk * D;
  const int nk = (int)(a.N - k0 < 16 * NT ? a.N - k0 : 16 * NT);

  // this wave's keys as column operands, and K^T for its head_dim tiles
  const int key = 16 * w + c;
  F kf[NK], vf[NK], kt[JD][KC];
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const bool ok = key < nk && 32 * i + 8 * g < D;
    const int64_t at = (key < nk ? key : 0) * rs + (32 * i + 8 * g < D ? 32 * i + 8 * g : 0);
    kf[i] = O::load(kp + at);
    vf[i] = O::load(vp + at);
    if (!ok) kf[i] = vf[i] = O::zero();
  }
#pragma unroll
  for (int i = 0; i < JD; ++i)
#pragma unroll
    for (int u = 0; u < KC; ++u) {
      const int d = 16 * (w + NT * i) + c;
      T e[8];
#pragma unroll
      for (int y = 0; y < 8; ++y) {
        const int kk = 32 * u + 16 * (y >> 2) + 4 * g + (y & 3);
        const bool ok = kk < nk && d < D;
        e[y] = kp[(kk < nk ? kk : 0) * rs + (d < D ? d : 0)];
        if (!ok) e[y] = static_cast<T>(0.0f);
      }
      kt[i][u] = __builtin_bit_cast(F, e);
    }
  int* flags = reinterpret_cast<int*>(lds + L::kFlag);  // [0], [1]: tiles in turn; [2]: the block's keys
  if (tid < 4) flags[tid] = 0;
  __syncthreads();
  if (a.causal) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NK; ++i) bad = bad || O::bad(kf[i]);
    if (bad) flags[2] = 1;
  }

  const int32_t* list = a.list + (int64_t)unit * a.N * a.S + item.y;
  const int64_t qbase = (int64_t)b * a.N * a.H + (int64_t)hk * a.G;
  const uint8_t* qp = static_cast<const uint8_t*>(a.q) + qbase * D * sizeof(T);
  const uint8_t* gp = static_cast<const uint8_t*>(a.g) + qbase * D * sizeof(T);
  const uint32_t qbytes = (uint32_t)(a.H * D) * sizeof(T), pbytes = (uint32_t)(a.G * D) * 4;
  uint8_t* part = reinterpret_cast<uint8_t*>(a.part + (int64_t)ug * a.N * a.S * a.G * D);
  const float* lse = a.lse_in + qbase;
  const float* dl = a.delta + qbase;

  // staging: chunk n of a thread is 8 elements of row (tid + n TH) / CPR; a
  // tile's pairs are read two tiles ahead, its rows one
  F sq[NC], sg[NC];
  int en[NC], est = 0;
  float s_lse = 0.0f, s_dl = 0.0f;
  int s_ent = 0, sown = 0;
  auto pair_of = [&](int rr) { return list[a.G == 1 ? rr : rr / a.G]; };
  auto head_of = [&](int rr) { return a.G == 1 ? 0 : rr % a.G; };
  // a row inside the block has keys that it may not see
  auto inside = [&](int e) { return a.causal && (e >> 6) - k0 < nk - 1; };
  auto pairs = [&](int r0) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int rr = r0 + (tid + n * TH) / CPR;
      en[n] = pair_of(rr < rows ? rr : rows - 1);
    }
    const int rt = r0 + (tid & (RT - 1));
    est = pair_of(rt < rows ? rt : rows - 1);
  };
  // no load and no store of the loop stands under a branch: rows past the end
  // load the last row, and store their dQ to a row that nothing reads (training
  // step of 2 x 8 heads on 4 of 4095 rows, head_dim 128: 517 -> 475 us)
  auto fetch = [&](int r0) {
    sown = 0;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int ch = tid + n * TH, rr = r0 + ch / CPR, d = (ch % CPR) * 8;
      const int hd = head_of(rr < rows ? rr : rows - 1) * D + (FULL || d < D ? d : 0);
      const uint64_t at = (uint64_t)(uint32_t)(en[n] >> 6) * qbytes + (uint32_t)hd * sizeof(T);
      sq[n] = O::load(reinterpret_cast<const T*>(qp + at));
      sg[n] = O::load(reinterpret_cast<const T*>(gp + at));
      sown |= inside(en[n]) << n;
    }
    const int rt = r0 + (tid & (RT - 1));
    const uint64_t at = (uint64_t)(uint32_t)(est >> 6) * (uint32_t)a.H + (uint32_t)head_of(rt < rows ? rt : rows - 1);
    s_lse = lse[at];
    s_dl = dl[at];
    s_ent = est;
  };

  f32x4 dv[ND], dk[ND];
#pragma unroll
  for (int j = 0; j < ND; ++j) dv[j] = dk[j] = f32x4{0, 0, 0, 0};
  int ex = kScaled<T> ? 100 : 0;  // dS are held times 2^ex
  const float sl2 = a.scale_log2;
  float* st_lse = reinterpret_cast<float*>(lds + L::kStat);
  float* st_dl = st_lse + RT;
  int* st_ent = reinterpret_cast<int*>(st_dl + RT);
  int* st_last = st_ent + RT;
  float* wmax = reinterpret_cast<float*>(lds + L::kMax);
  const int kabs = key < nk ? k0 + key : INT32_MAX;  // a row sees it if this is at most its last key

  if (rows > 0) {
    pairs(0);
    fetch(0);
    pairs(RT);
  }
  int turn = 0;
  for (int r0 = 0; r0 < rows; r0 += RT, turn ^= 1) {
    __syncthreads();  // the last tile has been read
    int sflag = 0;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int ch = tid + n * TH, row = ch / CPR, off = row * L::RS + (ch % CPR) * 8 * (int)sizeof(T);
      if (r0 + RT > rows || !FULL) {  // zeros past the end and past head_dim
        if (r0 + row >= rows || (ch % CPR) * 8 >= D) sq[n] = sg[n] = O::zero();
      }
      if (ch < RT * CPR) {
        *reinterpret_cast<F*>(lds + L::kQ + off) = sq[n];
        *reinterpret_cast<F*>(lds + L::kG + off) = sg[n];
        if ((sown >> n & 1) && (O::bad(sq[n]) || O::bad(sg[n]))) sflag |= 2;
      }
    }
    if (tid < RT) {
      st_lse[tid] = r0 + tid < rows ? s_lse : INFINITY;  // a row past the end has no weight
      st_dl[tid] = r0 + tid < rows ? s_dl : 0.0f;
      st_ent[tid] = s_ent;
      st_last[tid] = r0 + tid >= rows ? -1 : (a.causal ? s_ent >> 6 : INT32_MAX - 1);
      if (r0 + tid < rows && inside(s_ent)) sflag |= 1;
    }
    if (sflag) atomicOr(&flags[turn], sflag);
    if (tid == 0) flags[turn ^ 1] = 0;
    __syncthreads();
    const int fl = flags[turn];
    const bool slow = (fl & 1) && ((fl & 2) || flags[2]);
    if (r0 + RT < rows) {
      fetch(r0 + RT);
      pairs(r0 + 2 * RT);
    }

    int exs[RT / 32];
#pragma unroll
    for (int h = 0; h < RT / 32; ++h) {  // 32 rows at a time
      float p[2][4], ds[2][4];
      bool ok[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int ru = 32 * h + 16 * u;
        f32x4 s = f32x4{0, 0, 0, 0}, dp = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const uint8_t* at = lds + (ru + c) * L::RS + (32 * i + 8 * g) * (int)sizeof(T);
          s = O::mma(O::load(reinterpret_cast<const T*>(at + L::kQ)), kf[i], s);
          dp = O::mma(O::load(reinterpret_cast<const T*>(at + L::kG)), vf[i], dp);
        }
        settle(s);
        settle(dp);
        const float4 rl = *reinterpret_cast<const float4*>(st_lse + ru + 4 * g);
        const float4 rd = *reinterpret_cast<const float4*>(st_dl + ru + 4 * g);
        const int4 rq = *reinterpret_cast<const int4*>(st_last + ru + 4 * g);
        const float le[4] = {rl.x, rl.y, rl.z, rl.w}, de[4] = {rd.x, rd.y, rd.z, rd.w};
        const int last[4] = {rq.x, rq.y, rq.z, rq.w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          ok[u][y] = kabs <= last[y];
          const float pr = __builtin_amdgcn_exp2f(fmaf(s[y], sl2, -le[y]));
          ds[u][y] = ok[u][y] ? pr * (dp[y] - de[y]) : 0.0f;  // the scale is applied to the results
          p[u][y] = ok[u][y] ? pr * __builtin_amdgcn_exp2f(W::kBias) : 0.0f;
        }
      }
      if constexpr (kScaled<T>) {
        float mx = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int y = 0; y < 4; ++y) mx = fmaxf(mx, fabsf(ds[u][y]));
#pragma unroll
        for (int k = 32; k >= 1; k >>= 1) mx = fmaxf(mx, __shfl_xor(mx, k, 64));
        if (h) __syncthreads();  // the last maxima have been read
        if (lane == 0) wmax[w] = mx;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT; ++i) mx = fmaxf(mx, wmax[i]);
        if (mx > 0.0f) {
          const int e = min(14 - __builtin_amdgcn_frexp_expf(mx), 100);
          if (e < ex) {
            const float f = ldexpf(1.0f, e - ex);
#pragma unroll
            for (int j = 0; j < ND; ++j)
#pragma unroll
              for (int y = 0; y < 4; ++y) dk[j][y] *= f;
            ex = e;
          }
        }
        const float f = ldexpf(1.0f, ex);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int y = 0; y < 4; ++y) ds[u][y] *= f;
      }
      exs[h] = ex;
      W pw, sw;
      pw.set(p[0], p[1]);
      sw.set(ds[0], ds[1]);
      // dS [key][row] through LDS for dQ
#pragma unroll
      for (int pl = 0; pl < W::N; ++pl) {
        uint8_t* at = lds + L::kS + pl * L::kSPlane + key * L::SS + (32 * h + 4 * g) * (int)sizeof(T);
        if constexpr (sizeof(T) == 2) {
          *reinterpret_cast<uint2*>(at) = make_uint2(sw.w[pl].x, sw.w[pl].y);
          *reinterpret_cast<uint2*>(at + 32) = make_uint2(sw.w[pl].z, sw.w[pl].w);
        } else {
          *reinterpret_cast<float4*>(at) = make_float4(ds[0][0], ds[0][1], ds[0][2], ds[0][3]);
          *reinterpret_cast<float4*>(at + 64) = make_float4(ds[1][0], ds[1][1], ds[1][2], ds[1][3]);
        }
      }
      if (__builtin_expect(slow, 0)) {
        // a row's infinity or NaN must not reach keys that it does not see
        for (int rr = 0; rr < 32; ++rr) {
          float pk = 0.0f, dk1 = 0.0f;
          int okk = 0;
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (u == rr >> 4 && y == (rr & 3)) pk = p[u][y], dk1 = ds[u][y], okk = ok[u][y];
          const int src = c + 16 * ((rr & 15) >> 2);
          pk = __shfl(pk, src, 64);
          dk1 = __shfl(dk1, src, 64);
          okk = __shfl(okk, src, 64);
          const T* qr = reinterpret_cast<const T*>(lds + L::kQ + (32 * h + rr) * L::RS);
          const T* gr = reinterpret_cast<const T*>(lds + L::kG + (32 * h + rr) * L::RS);
          if (okk)
#pragma unroll
            for (int j = 0; j < ND; ++j)
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                dv[j][y] += pk * (float)gr[16 * j + 4 * g + y];
                dk[j][y] += dk1 * (float)qr[16 * j + 4 * g + y];
              }
        }
      } else {
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          F gt, qt;
          if constexpr (sizeof(T) == 2) {
            const uint8_t* at = lds + (32 * h + 4 * g + (c >> 2)) * L::RS + (16 * j + 4 * (c & 3)) * 2;
            const uint2 g0 = tr_read(at + L::kG), g1 = tr_read(at + L::kG + 16 * L::RS);
            const uint2 q0 = tr_read(at + L::kQ), q1 = tr_read(at + L::kQ + 16 * L::RS);
            gt = make_uint4(g0.x, g0.y, g1.x, g1.y);
            qt = make_uint4(q0.x, q0.y, q1.x, q1.y);
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              const uint8_t* at = lds + (32 * h + 16 * (y >> 2) + 4 * g + (y & 3)) * L::RS + (16 * j + c) * 4;
              gt.v[y] = *reinterpret_cast<const float*>(at + L::kG);
              qt.v[y] = *reinterpret_cast<const float*>(at + L::kQ);
            }
          }
#pragma unroll
          for (int pl = W::N - 1; pl >= 0; --pl) {
            dv[j] = O::mma(gt, pw.w[pl], dv[j]);
            dk[j] = O::mma(qt, sw.w[pl], dk[j]);
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < RT / 16; ++u) {
      const int rr = r0 + 16 * u + c;
      const float back = kScaled<T> ? ldexpf(1.0f, -exs[u / 2]) : 1.0f;
      f32x4 dq[JD];
#pragma unroll
      for (int i = 0; i < JD; ++i) dq[i] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int v = 0; v < KC; ++v) {
#pragma unroll
        for (int pl = W::N - 1; pl >= 0; --pl) {
          F sf;
          if constexpr (sizeof(T) == 2) {
            const uint8_t* at =
                lds + L::kS + pl * L::kSPlane + (32 * v + 4 * g + (c >> 2)) * L::SS + (16 * u + 4 * (c & 3)) * 2;
            const uint2 s0 = tr_read(at);
            uint2 s1 = make_uint2(0, 0);
            if constexpr (NT > 1) s1 = tr_read(at + 16 * L::SS);
            sf = make_uint4(s0.x, s0.y, s1.x, s1.y);
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y)
              sf.v[y] = NT > 1 || y < 4 ? *reinterpret_cast<const float*>(
                                              lds + L::kS + (32 * v + 16 * (y >> 2) + 4 * g + (y & 3)) * L::SS + (16 * u + c) * 4)
                                        : 0.0f;
          }
#pragma unroll
          for (int i = 0; i < JD; ++i) dq[i] = O::mma(kt[i][v], sf, dq[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < JD; ++i) settle(dq[i]);
      if (__builtin_expect(slow, 0)) {
#pragma unroll
        for (int i = 0; i < JD; ++i) dq[i] = f32x4{0, 0, 0, 0};
        for (int kk = 0; kk < nk; ++kk) {
          float d1 = 0.0f;
#pragma unroll
          for (int pl = W::N - 1; pl >= 0; --pl)
            d1 += (float)*reinterpret_cast<const T*>(lds + L::kS + pl * L::kSPlane + kk * L::SS + (16 * u + c) * (int)sizeof(T));
          if (k0 + kk > st_last[16 * u + c]) continue;
#pragma unroll
          for (int i = 0; i < JD; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int d = 16 * (w + NT * i) + 4 * g + y;
              if (d < D) dq[i][y] += d1 * (float)kp[kk * rs + d];
            }
        }
      }
      const int e = st_ent[16 * u + c];
      float* po = reinterpret_cast<float*>(part + (uint64_t)(__umul24(e >> 6, a.S) + (e & 63)) * pbytes) +
                  head_of(rr < rows ? rr : rows - 1) * D;
      po = rr < rows ? po : a.unread;
#pragma unroll
      for (int i = 0; i < JD; ++i) {
        const int d = 16 * (w + NT * i) + 4 * g;
        if ((FULL && ND % NT == 0) || d < D)
          __builtin_nontemporal_store(f32x4{dq[i][0] * back, dq[i][1] * back, dq[i][2] * back, dq[i][3] * back},
                                      reinterpret_cast<f32x4*>(po + d));
      }
    }
  }
  // dK, dV: the only item of its block stores them, others leave parts
  const bool single = a.blk_items[(int64_t)unit * a.nb + blk].y == 1;
  const float fv = __builtin_amdgcn_exp2f(-W::kBias), fk = (kScaled<T> ? ldexpf(1.0f, -ex) : 1.0f) * a.scale;
  if (key >= nk) return;
#pragma unroll
  for (int j = 0; j < ND; ++j) {
    const int d = 16 * j + 4 * g;
    if (d >= D) continue;
    if (single) {
      T k4[4], v4[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        k4[y] = static_cast<T>(dk[j][y] * fk);
        v4[y] = static_cast<T>(dv[j][y] * fv);
      }
      const int64_t at = ((int64_t)b * a.N + k0 + key) * rs + hk * D + d;
      T* ok = static_cast<T*>(a.dk) + at;
      T* ov = static_cast<T*>(a.dv) + at;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(ok) = *reinterpret_cast<const uint2*>(k4);
        *reinterpret_cast<uint2*>(ov) = *reinterpret_cast<const uint2*>(v4);
      } else {
        *reinterpret_cast<uint4*>(ok) = *reinterpret_cast<const uint4*>(k4);
        *reinterpret_cast<uint4*>(ov) = *reinterpret_cast<const uint4*>(v4);
      }
    } else {
      float* pk = a.part_kv + (((int64_t)ug * a.max_items + slot_item) * 2 * a.BS + key) * D + d;
      *reinterpret_cast<float4*>(pk) = make_float4(dk[j][0] * fk, dk[j][1] * fk, dk[j][2] * fk, dk[j][3] * fk);
      *reinterpret_cast<float4*>(pk + (int64_t)a.BS * D) =
          make_float4(dv[j][0] * fv, dv[j][1] * fv, dv[j][2] * fv, dv[j][3] * fv);
    }
  }
}

// The parts of a block with more than one item, added in list order by
// kKvParts workgroups.
constexpr int kKvParts = 8;

template <typename T>
__global__ __launch_bounds__(256) void join_kv_kernel(Args a) {
  const uint32_t x = blockIdx.x / (uint32_t)kKvParts;
  const int ug = x / (uint32_t)a.nb, blk = x % (uint32_t)a.nb, unit = a.unit0 + ug;
  const int2 bi = a.blk_items[(int64_t)unit * a.nb + blk];
  if (bi.y == 1) return;
  const int b = unit / a.Hkv, hk = unit % a.Hkv, D = a.D, q4 = D >> 2;
  const int64_t k0 = (int64_t)blk * a.BS, rs = (int64_t)a.Hkv * D;
  const int nk = (int)(a.N - k0 < a.BS ? a.N - k0 : a.BS);
  const float* p0 = a.part_kv + ((int64_t)ug * a.max_items + bi.x) * 2 * a.BS * D;
  for (int e = blockIdx.x % (uint32_t)kKvParts * 256 + threadIdx.x; e < 2 * a.BS * q4; e += 256 * kKvParts) {
    const int m = e / (a.BS * q4), r = e - m * a.BS * q4, key = r / q4, d = 4 * (r - key * q4);
    if (key >= nk) continue;
    float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int i = 0; i < bi.y; ++i) {
      const float4 y = *reinterpret_cast<const float4*>(p0 + ((int64_t)(2 * i + m) * a.BS + key) * D + d);
      s.x += y.x, s.y += y.y, s.z += y.z, s.w += y.w;
    }
    T t[4] = {static_cast<T>(s.x), static_cast<T>(s.y), static_cast<T>(s.z), static_cast<T>(s.w)};
    T* o = static_cast<T*>(m ? a.dv : a.dk) + (int64_t)b * a.N * rs + (k0 + key) * rs + hk * D + d;
    if constexpr (sizeof(T) == 2)
      *reinterpret_cast<uint2*>(o) = *reinterpret_cast<const uint2*>(t);
    else
      *reinterpret_cast<uint4*>(o) = *reinterpret_cast<const uint4*>(t);
  }
}

}  // namespace ma_selected
