// paged_kernel.h -- kernels of the paged key/value cache: append with the
// position rotation, attention of one token per stream, and the selection of
// pages from their key sums.
#pragma once

#include "attn_planes.h"
#include "device_common.h"
#include "top_select.h"

namespace ma_paged {

using namespace ma_dev;

// ---------------------------------------------------------------- append
//
// y_a = x_a cos t - x_b sin t, y_b = x_a sin t + x_b cos t with t = position *
// inv_freq, all in float64: a far position's angle needs it, and the page sums
// add up the rounded keys, so a key next to a rounding border has to fall the
// same way whoever computes it.  The angles of a tile of tokens are computed
// once into LDS and serve every query and key head.
//
// One workgroup takes one page's worth of positions of one stream, so that with
// page sums it owns the page: after its stores it reads the page's stored
// keys [0, end) back (cache-hot) and adds them in slot order classes.  The sum
// depends on the page's contents alone, not on the calls that filled it: a
// stream that is set back and appended to again needs no correction.
//
// Bound by bytes on a prompt: 4 x 8191 tokens (three quarters stored), 8 heads of
// 64, f16 take 33 us, 169 MB at 5.0 TB/s; a single token's launch 6 us.

struct AppendArgs {
  const void* k;
  const void* v;
  const void* q;
  void* qo;
  void* ck;
  void* cv;
  float* sums;
  const int32_t* table;
  const int32_t* start;
  const int32_t* counts;
  const double* freq;
  int64_t n;        // new tokens per stream
  int64_t width;    // pages per stream
  int64_t pages;    // pages of the cache
  int32_t page;     // tokens per page
  int32_t step;     // positions per workgroup
  int32_t H, Hkv, D, R, inter;
  int32_t wgs;      // workgroups per stream
};

constexpr int kAppendThreads = 512;
constexpr int kSumParts = kAppendThreads / 32;  // slot classes of a page sum
constexpr int kAppendTile = 16;  // tokens whose angles are in LDS at once

// Eight elements as float32 values or raw bits.
template <typename T>
struct Vec8 {
  T x[8];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p);
    } else {
      reinterpret_cast<uint4*>(x)[0] = reinterpret_cast<const uint4*>(p)[0];
      reinterpret_cast<uint4*>(x)[1] = reinterpret_cast<const uint4*>(p)[1];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(x);
    } else {
      reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<const uint4*>(x)[0];
      reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<const uint4*>(x)[1];
    }
  }
};

// Through float32, as torch converts float64 (the compiler would fold the two
// conversions to f16 into one).
template <typename T>
__device__ __forceinline__ T round_to(double y) {
  float f = static_cast<float>(y);
  asm volatile("" : "+v"(f));
  return static_cast<T>(f);
}

// Rotates the row at src (head_dim D, R of it rotated) into dst, one unit of
// the row per call: units [0, R/16) are 16 rotated elements each (two chunks
// that hold each other's partners), the rest copy 8.
template <typename T>
__device__ __forceinline__ void rotate_unit(const T* src, T* dst, int u, int R, int inter, const double2* cs) {
  const int nr = R >> 4;
  Vec8<T> a, b;
  if (u >= nr) {
    const int o = R + 8 * (u - nr);
    a.load(src + o);
    a.store(dst + o);
    return;
  }
  if (inter) {
    a.load(src + 16 * u);
    b.load(src + 16 * u + 8);
    const double2* c = cs + 8 * u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double x0 = (double)(float)a.x[2 * j], x1 = (double)(float)a.x[2 * j + 1];
      a.x[2 * j] = round_to<T>(x0 * c[j].x - x1 * c[j].y);
      a.x[2 * j + 1] = round_to<T>(x0 * c[j].y + x1 * c[j].x);
      const double z0 = (double)(float)b.x[2 * j], z1 = (double)(float)b.x[2 * j + 1];
      b.x[2 * j] = round_to<T>(z0 * c[4 + j].x - z1 * c[4 + j].y);
      b.x[2 * j + 1] = round_to<T>(z0 * c[4 + j].y + z1 * c[4 + j].x);
    }
    a.store(dst + 16 * u);
    b.store(dst + 16 * u + 8);
    return;
  }
  a.load(src + 8 * u);
  b.load(src + (R >> 1) + 8 * u);
  const double2* c = cs + 8 * u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const double x0 = (double)(float)a.x[j], x1 = (double)(float)b.x[j];
    a.x[j] = round_to<T>(x0 * c[j].x - x1 * c[j].y);
    b.x[j] = round_to<T>(x0 * c[j].y + x1 * c[j].x);
  }
  a.store(dst + 8 * u);
  b.store(dst + (R >> 1) + 8 * u);
}

template <typename T>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int32_t s_slot[kAppendTile];
  double2* cs = reinterpret_cast<double2*>(lds);  // [kAppendTile][R / 2]
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x / (uint32_t)a.wgs;
  const int w = blockIdx.x % (uint32_t)a.wgs;
  const int64_t s0 = a.start[b] > 0 ? a.start[b] : 0;
  int64_t cnt = a.counts ? a.counts[b] : a.n;
  cnt = cnt < 0 ? 0 : (cnt > a.n ? a.n : cnt);
  const int64_t base = a.sums ? s0 / a.page * a.page : s0;
  int64_t p0 = base + (int64_t)w * a.step, p1 = p0 + a.step;
  if (p0 < s0) p0 = s0;
  if (p1 > s0 + a.n) p1 = s0 + a.n;
  if (p0 >= p1) return;
  const int D = a.D, R = a.R, half = R >> 1;
  const int upr = (R >> 4) + ((D - R) >> 3);  // units per rotated row
  const int nk = a.Hkv * upr, nv = a.Hkv * (D >> 3), nq = a.q ? a.H * upr : 0;
  const T* kin = static_cast<const T*>(a.k);
  const T* vin = static_cast<const T*>(a.v);
  const T* qin = static_cast<const T*>(a.q);
  T* ck = static_cast<T*>(a.ck);
  T* cv = static_cast<T*>(a.cv);
  T* qo = static_cast<T*>(a.qo);
  const int nr = nk + nq;
  const int tv = tid / nv, uv = tid - tv * nv, sv = kAppendThreads / nv;
  const int tr = tid / nr, ur = tid - tr * nr, sr = kAppendThreads / nr;
  const uint32_t kvrow = (uint32_t)(a.Hkv * D);
  for (int64_t t0 = p0; t0 < p1; t0 += kAppendTile) {
    const int nt = (int)(p1 - t0 < kAppendTile ? p1 - t0 : kAppendTile);
    __syncthreads();  // the last tile's angles and slots have been read
    if (tid < nt) {
      // where the token is stored; -1: behind the count, the table or the cache
      const int64_t pos = t0 + tid, l = pos / a.page;
      int32_t slot = -1;
      if (pos - s0 < cnt && l < a.width) {
        const int32_t ph = a.table[b * a.width + l];
        if (ph >= 0 && ph < a.pages) slot = ph * a.page + (int32_t)(pos - l * a.page);
      }
      s_slot[tid] = slot;
    }
    if (half) {
      for (int e = tid; e < nt * half; e += kAppendThreads) {
        const int t = e / half, j = e - t * half;
        double s, c;
        sincos((double)(t0 + t) * a.freq[j], &s, &c);
        cs[t * half + j] = make_double2(c, s);
      }
    }
    __syncthreads();
    const uint32_t row0 = (uint32_t)(t0 - s0);
    // values: chunk u of token t, a step of kAppendThreads chunks at a time (the
    // heads' values are one run of elements)
    for (int t = tv, u = uv; t < nt; t += sv, u += kAppendThreads - sv * nv) {
      if (u >= nv) {
        u -= nv;
        if (++t >= nt) break;
      }
      const int32_t slot = s_slot[t];
      const uint64_t row = (uint64_t)b * (uint32_t)a.n + (row0 + t);
      Vec8<T> x;
      x.load(vin + row * kvrow + 8 * u);
      if (slot >= 0) x.store(cv + (uint64_t)(uint32_t)slot * kvrow + 8 * u);
    }
    // keys and queries, which differ in their addresses alone: lanes of one wave
    // take the same path
    for (int t = tr, u = ur; t < nt; t += sr, u += kAppendThreads - sr * nr) {
      if (u >= nr) {
        u -= nr;
        if (++t >= nt) break;
      }
      const int32_t slot = s_slot[t];
      const uint64_t row = (uint64_t)b * (uint32_t)a.n + (row0 + t);
      const bool isq = u >= nk;
      if (!isq && slot < 0) continue;
      const uint32_t v = (uint32_t)(isq ? u - nk : u), h = v / (uint32_t)upr;
      const uint64_t qo_at = row * (uint32_t)(a.H * D) + h * D, ki = row * kvrow + h * D;
      const T* src = isq ? qin + qo_at : kin + ki;
      T* dst = isq ? qo + qo_at : ck + (uint64_t)(uint32_t)slot * kvrow + h * D;
      rotate_unit<T>(src, dst, (int)(v - h * upr), R, a.inter, cs + t * half);
    }
  }
  if (!a.sums) return;
  // the page's stored keys, back from the cache: thread (r, c) adds every
  // kSumParts-th slot of 8 elements, and the parts are joined in order
  const int64_t last = p1 < s0 + cnt ? p1 : s0 + cnt;
  const int64_t l = p0 / a.page;
  if (last <= p0 || l >= a.width) return;
  const int32_t ph = a.table[b * a.width + l];
  if (ph < 0 || ph >= a.pages) return;
  const int end = (int)(last - l * a.page);
  __syncthreads();  // every store of this workgroup is visible to it; the angles are free
  float* part = reinterpret_cast<float*>(lds);  // [kSumParts][32 chunks][8]
  const int chunks = a.Hkv * (D >> 3);
  const int r = tid >> 5, c0 = tid & 31;
  for (int cb = 0; cb < chunks; cb += 32) {
    const int c = cb + c0;
    float acc[8] = {};
    if (c < chunks) {
      const T* p = ck + (int64_t)ph * a.page * a.Hkv * D + 8 * c;
#pragma unroll 4
      for (int s = r; s < end; s += kSumParts) {
        Vec8<T> x;
        x.load(p + (int64_t)s * a.Hkv * D);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += (float)x.x[j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) part[tid * 8 + j] = acc[j];
    __syncthreads();
    const int e = tid;  // 32 chunks x 8 elements
    if (e < 256 && cb * 8 + e < chunks * 8) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < kSumParts; ++i) s += part[i * 256 + e];
      a.sums[(int64_t)ph * a.Hkv * D + cb * 8 + e] = s;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- decode
//
// One wave streams 32 keys a step.  S^T = K Q^T puts a head in each MFMA
// column and four keys of each 16-key tile in each lane, which is the operand
// layout of O^T = V^T P^T for the same keys: the weights never leave their
// lane, the running maximum and sum are per lane, and there is no LDS in the
// loop.  Queries that share a key/value head share its columns, so a step's
// keys and values are read once for up to 16 of them.  The values' operand
// (eight keys of one head_dim element) is two-by-two permutes of eight rows
// that the lane loads itself.
//
// Bound by the cache's bytes: one step's loads are in flight while the last is
// computed, and the token range is split over enough workgroups to fill the
// card; their (maximum, sum, output) partials are joined by a second kernel.
// One stream of 65536 tokens, 8 heads of 64, f16: 26 us (5.2 TB/s) and 4.2 for
// the join; 32 streams of up to 8192, 2 heads of 128, bf16: 36 us (5.4 TB/s).

struct DecodeArgs {
  const void* q;
  const void* ck;
  const void* cv;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* pages;  // listed pages, or null
  void* out;
  float* lse;
  float* part_o;   // [B * H][nsplit][D]
  float* part_ml;  // [B * H][nsplit][2]
  int64_t num_pages;
  int32_t width, page, H, Hkv, G, gt, D, S, nsplit;
  int32_t windowed;
  int64_t left, nglobal;
  float scale_log2;
};

constexpr int kDecWaves = 4;

// The keys a tile of 16 covers: the token's slot in the cache and the valid
// part [lo, hi) of the 16; hi <= lo: none.
struct Tile {
  int32_t tok;
  int32_t rng;  // lo | hi << 8
};

__device__ __forceinline__ Tile make_tile(const DecodeArgs& a, int64_t b, int64_t base, int64_t seg_lo,
                                          int64_t seg_hi) {
  Tile t{0, 0};
  if (seg_hi <= base || seg_lo >= base + 16) return t;
  const uint32_t l = (uint32_t)base / (uint32_t)a.page;  // base < seg_hi <= width * page < 2^31
  if (l >= (uint32_t)a.width) return t;
  const int32_t ph = a.table[b * a.width + l];
  if (ph < 0 || ph >= a.num_pages) return t;
  t.tok = ph * a.page + (int32_t)((uint32_t)base - l * (uint32_t)a.page);
  const int lo = seg_lo > base ? (int)(seg_lo - base) : 0;
  const int hi = seg_hi < base + 16 ? (int)(seg_hi - base) : 16;
  t.rng = lo | hi << 8;
  return t;
}

// A stream's key set as a list of 16-key tiles.
struct KeySet {
  int64_t len, ws, ng, wbase;
  int32_t ntg, total, tpp;
  int32_t ent;  // listed pages: lane l has entry l, -1 where it is skipped
  bool listed;

  __device__ __forceinline__ void init(const DecodeArgs& a, int64_t b, int hk, int lane) {
    listed = a.pages != nullptr;
    ent = -1;
    if (listed && lane < a.S) ent = a.pages[(b * a.Hkv + hk) * a.S + lane];
    len = a.lengths[b];
    const int64_t cap = (int64_t)a.width * a.page;
    len = len < 0 ? 0 : (len > cap ? cap : len);
    tpp = a.page >> 4;
    ws = 0;
    ng = 0;
    if (listed) {
      for (int j = 0; j + 1 < a.S; ++j) {  // repeats count once
        const int o = __builtin_amdgcn_readlane(ent, j);
        if (j < lane && o == ent) ent = -1;
      }
      total = len > 0 ? a.S * tpp : 0;
      return;
    }
    if (a.windowed) {
      ws = len - 1 - a.left;
      ws = ws < 0 ? 0 : ws;
      ng = a.nglobal < ws ? a.nglobal : ws;
    }
    wbase = ws & ~15ll;
    ntg = (int32_t)((ng + 15) >> 4);
    total = ntg + (int32_t)((len - wbase + 15) >> 4);
    if (len == 0) total = 0;
  }

  // Tile t of the lane; every lane of the wave calls it.
  __device__ __forceinline__ Tile tile(const DecodeArgs& a, int64_t b, int32_t t, bool in) const {
    if (listed) {
      const int e = in ? t / tpp : 0;
      const int32_t p = __shfl(ent, e, 64);
      if (!in || p < 0) return Tile{0, 0};
      return make_tile(a, b, (int64_t)p * a.page + (t - e * tpp) * 16, 0, len);
    }
    if (!in) return Tile{0, 0};
    if (t < ntg) return make_tile(a, b, (int64_t)t * 16, 0, ng);
    return make_tile(a, b, wbase + (int64_t)(t - ntg) * 16, ws, len);
  }
};

// Operands of one 16-bit or float32 key/value step of 32 keys (two tiles).
template <typename T, int DP, bool FULL>
struct Step {
  static constexpr bool k16 = sizeof(T) == 2;
  static constexpr int NK = k16 ? DP / 32 : DP / 16;  // 16-byte key loads per tile
  static constexpr int VPL = DP / 16;                 // value elements per lane and key
  static constexpr int VW = VPL * (int)sizeof(T) / 4; // 32-bit words of them
  uint4 k[2][NK];
  uint32_t v[2][4][VW];
  int32_t rng[2];

  __device__ __forceinline__ void load(const DecodeArgs& a, Tile t0, Tile t1, int hk, int c, int g) {
    const Tile t[2] = {t0, t1};
    const int64_t row = (int64_t)a.Hkv * a.D;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      rng[u] = t[u].rng;
      const T* kb = static_cast<const T*>(a.ck) + (int64_t)t[u].tok * row + hk * a.D;
      const T* vb = static_cast<const T*>(a.cv) + (int64_t)t[u].tok * row + hk * a.D;
      constexpr int EPL = k16 ? 8 : 4;  // elements of a 16-byte load
#pragma unroll
      for (int x = 0; x < NK; ++x) {
        const int d = (4 * x + g) * EPL;
        const bool ok = FULL || d < a.D;
        k[u][x] = *reinterpret_cast<const uint4*>(kb + (uint32_t)(c * (int)row + (ok ? d : 0)));
        if (!ok) k[u][x] = make_uint4(0, 0, 0, 0);
      }
      const int dv = (FULL || c * VPL < a.D) ? c * VPL : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(vb + (uint32_t)((4 * g + i) * (int)row + dv));
        if constexpr (VW == 1) {
          v[u][i][0] = p[0];
        } else if constexpr (VW == 2) {
          const uint2 x = *reinterpret_cast<const uint2*>(p);
          v[u][i][0] = x.x;
          v[u][i][1] = x.y;
        } else {
#pragma unroll
          for (int w = 0; w < VW; w += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + w);
            v[u][i][w] = x.x;
            v[u][i][w + 1] = x.y;
            v[u][i][w + 2] = x.z;
            v[u][i][w + 3] = x.w;
          }
        }
      }
    }
  }
};

// Waves per SIMD that the registers are budgeted for; two or more also keep the
// products out of the accumulation registers.
template <typename T, int DP>
constexpr int kDecOcc = DP * (int)sizeof(T) > 256 ? 1 : (DP * (int)sizeof(T) > 128 ? 2 : 3);

template <typename T, int DP, bool FULL>
__global__ __launch_bounds__(64 * kDecWaves, (kDecOcc<T, DP>)) void decode_kernel(DecodeArgs a) {
  using St = Step<T, DP, FULL>;
  constexpr bool k16 = sizeof(T) == 2;
  constexpr int NK = St::NK, VPL = St::VPL;
  __shared__ float s_o[kDecWaves][16][DP + 4];
  __shared__ float s_m[kDecWaves][16], s_l[kDecWaves][16];
  __shared__ int s_any[kDecWaves];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, c = lane & 15, g = lane >> 4;
  uint32_t x = blockIdx.x;
  const int sp = x % (uint32_t)a.nsplit;
  x /= (uint32_t)a.nsplit;
  const int gt = x % (uint32_t)a.gt;
  x /= (uint32_t)a.gt;
  const int hk = x % (uint32_t)a.Hkv;
  const int64_t b = x / (uint32_t)a.Hkv;
  const int gn = a.G - 16 * gt < 16 ? a.G - 16 * gt : 16;  // heads of this workgroup
  const int h0 = hk * a.G + 16 * gt;

  KeySet ks;
  ks.init(a, b, hk, lane);
  const int steps = (ks.total + 1) >> 1;
  const int per = (steps + a.nsplit - 1) / a.nsplit;
  const int s0 = sp * per;
  const int s1 = s0 + per < steps ? s0 + per : steps;

  // queries: column c is head h0 + c
  uint4 qf[NK];
  {
    const T* qp = static_cast<const T*>(a.q) + ((int64_t)b * a.H + h0 + (c < gn ? c : 0)) * a.D;
    constexpr int EPL = k16 ? 8 : 4;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int d = (4 * i + g) * EPL;
      const bool ok = (FULL || d < a.D) && c < gn;
      qf[i] = *reinterpret_cast<const uint4*>(qp + (ok ? d : 0));
      if (!ok) qf[i] = make_uint4(0, 0, 0, 0);
    }
  }

  f32x4 acc[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) acc[j] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  int any = 0;
  const float sl2 = a.scale_log2;
  constexpr float kBias = WeightPlanes<T>::kBias;

  auto compute = [&](const St& st) {
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        if constexpr (k16) {
          s[u] = Mma<T>::x32(st.k[u][i], qf[i], s[u]);
        } else {
          s[u] = mfma_f32(__uint_as_float(st.k[u][i].x), __uint_as_float(qf[i].x), s[u]);
          s[u] = mfma_f32(__uint_as_float(st.k[u][i].y), __uint_as_float(qf[i].y), s[u]);
          s[u] = mfma_f32(__uint_as_float(st.k[u][i].z), __uint_as_float(qf[i].z), s[u]);
          s[u] = mfma_f32(__uint_as_float(st.k[u][i].w), __uint_as_float(qf[i].w), s[u]);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[u][r] *= sl2;
    }
    uint32_t v[2][4][St::VW];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int y = 0; y < St::VW; ++y) v[u][i][y] = st.v[u][i][y];
    if (st.rng[0] != (16 << 8) || st.rng[1] != (16 << 8)) {
      // rows outside the set may hold anything: no score, and zero values
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int lo = st.rng[u] & 255, hi = st.rng[u] >> 8;
        any |= hi > lo;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool ok = 4 * g + r >= lo && 4 * g + r < hi;
          s[u][r] = ok ? s[u][r] : -INFINITY;
#pragma unroll
          for (int y = 0; y < St::VW; ++y) v[u][r][y] = ok ? v[u][r][y] : 0u;
        }
      }
    } else {
      any = 1;
    }
    float mt = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mt = col_max(mt);
    const float mn = fmaxf(m, mt);
    const float mu = mn == -INFINITY ? 0.0f : mn;
    const float al = m == mn ? 1.0f : __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    float p[2][4];
    float ps = 0.0f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[u][r] = __builtin_amdgcn_exp2f(s[u][r] - mu + kBias);
        ps += p[u][r];
      }
    l = l * al + ps;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[j][r] *= al;
    if constexpr (k16) {
      WeightPlanes<T> pp;
      pp.set(p[0], p[1]);
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        // eight keys' element j: halves (j & 1) of word j / 2, two keys a word
        constexpr uint32_t kSel[2] = {0x05040100u, 0x07060302u};
        uint4 vf;
        vf.x = __builtin_amdgcn_perm(v[0][1][j / 2], v[0][0][j / 2], kSel[j & 1]);
        vf.y = __builtin_amdgcn_perm(v[0][3][j / 2], v[0][2][j / 2], kSel[j & 1]);
        vf.z = __builtin_amdgcn_perm(v[1][1][j / 2], v[1][0][j / 2], kSel[j & 1]);
        vf.w = __builtin_amdgcn_perm(v[1][3][j / 2], v[1][2][j / 2], kSel[j & 1]);
#pragma unroll
        for (int pl = WeightPlanes<T>::N - 1; pl >= 0; --pl) acc[j] = Mma<T>::x32(vf, pp.w[pl], acc[j]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < VPL; ++j) acc[j] = mfma_f32(__uint_as_float(v[u][r][j]), p[u][r], acc[j]);
    }
  };

  // this wave's steps: s0 + w, s0 + w + 4, ...; the tiles of 32 of them are
  // worked out by the lanes at once
  const int mine = s1 - s0 - w > 0 ? (s1 - s0 - w + kDecWaves - 1) / kDecWaves : 0;
  Tile td{0, 0};
  auto tiles = [&](int it) {
    const int step = s0 + w + kDecWaves * (it + (lane >> 1));
    const int t = 2 * step + (lane & 1);
    td = ks.tile(a, b, t, step < s1 && t < ks.total);
  };
  auto pick = [&](int i) {
    return Tile{__builtin_amdgcn_readlane(td.tok, i), __builtin_amdgcn_readlane(td.rng, i)};
  };
  if (mine > 0) {
    St A, B;
    tiles(0);
    A.load(a, pick(0), pick(1), hk, c, g);
    for (int it = 0; it < mine; it += 2) {
      const int i1 = (it + 1) & 31;
      B.load(a, pick(2 * i1), pick(2 * i1 + 1), hk, c, g);  // an invalid step reads slot 0, unused
      compute(A);
      if (it + 1 >= mine) break;
      if (((it + 2) & 31) == 0) tiles(it + 2);
      const int i2 = (it + 2) & 31;
      A.load(a, pick(2 * i2), pick(2 * i2 + 1), hk, c, g);
      compute(B);
    }
  }
  l = col_sum(l);

  // join the four waves
#pragma unroll
  for (int j = 0; j < VPL; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) s_o[w][c][(4 * g + r) * VPL + j] = acc[j][r];
  if (g == 0) {
    s_m[w][c] = m;
    s_l[w][c] = l;
  }
  if (lane == 0) s_any[w] = any;
  __syncthreads();
  const int anyw = s_any[0] | s_any[1] | s_any[2] | s_any[3];
  for (int e = tid; e < gn * a.D; e += 64 * kDecWaves) {
    const int h = e / a.D, d = e - h * a.D;
    const float M = fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h]));
    const float mu = M == -INFINITY ? 0.0f : M;
    float o = 0.0f, lt = 0.0f;
#pragma unroll
    for (int i = 0; i < kDecWaves; ++i) {
      const float f = __builtin_amdgcn_exp2f(s_m[i][h] - mu);
      o += f * s_o[i][h][d];
      lt += f * s_l[i][h];
    }
    const int64_t row = b * a.H + h0 + h;
    if (a.nsplit == 1) {
      static_cast<T*>(a.out)[row * a.D + d] = static_cast<T>(anyw ? o / lt : 0.0f);
      if (a.lse && d == 0) a.lse[row] = anyw ? M + (__log2f(lt) - kBias) : -INFINITY;
    } else {
      a.part_o[(row * a.nsplit + sp) * a.D + d] = o;
      if (d == 0) {
        a.part_ml[(row * a.nsplit + sp) * 2] = M;
        a.part_ml[(row * a.nsplit + sp) * 2 + 1] = anyw ? lt : -1.0f;  // -1: no key here
      }
    }
  }
}

// Joins the splits of one (stream, head): o = sum 2^(m_s - M) o_s / sum 2^(m_s - M) l_s.
// 1024 / DT groups of DT threads take every group-th split; a thread's first
// eight outputs are under way before the weights are known.
constexpr int kJoinThreads = 1024;
constexpr int kMaxSplit = 256;

template <typename T, int DT>
__global__ __launch_bounds__(kJoinThreads) void decode_join_kernel(DecodeArgs a) {
  constexpr int NG = kJoinThreads / DT;
  __shared__ float s_f[kMaxSplit];
  __shared__ float s_red[kJoinThreads];
  __shared__ float s_m[kMaxSplit / 64], s_l[kMaxSplit / 64];
  __shared__ int s_any[kMaxSplit / 64];
  const int tid = threadIdx.x, w = tid >> 6;
  const int64_t row = blockIdx.x;
  const float* ml = a.part_ml + row * a.nsplit * 2;
  const int D = a.D, d = tid % DT, gr = tid / DT;
  const float* po = a.part_o + row * a.nsplit * D + (d < D ? d : 0);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = gr + i * NG < a.nsplit ? po[(int64_t)(gr + i * NG) * D] : 0.0f;
  // statistics: thread s < 256 has split s
  float M = -INFINITY, ls = -1.0f;
  if (tid < kMaxSplit) {
    if (tid < a.nsplit) {
      M = ml[2 * tid];
      ls = ml[2 * tid + 1];
    }
    float mw = M;
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) mw = fmaxf(mw, __shfl_xor(mw, k, 64));
    const bool any = __ballot(ls != -1.0f) != 0;  // -1: the split has no key
    if ((tid & 63) == 0) {
      s_m[w] = mw;
      s_any[w] = any;
    }
  }
  __syncthreads();
  const float Mt = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float mu = Mt == -INFINITY ? 0.0f : Mt;
  const bool any = (s_any[0] | s_any[1] | s_any[2] | s_any[3]) != 0;
  if (tid < kMaxSplit) {
    const float f = ls == -1.0f ? 0.0f : __builtin_amdgcn_exp2f(M - mu);
    s_f[tid] = ls == -1.0f ? -1.0f : f;
    float l = ls == -1.0f ? 0.0f : f * ls;
#pragma unroll
    for (int k = 32; k >= 1; k >>= 1) l += __shfl_xor(l, k, 64);
    if ((tid & 63) == 0) s_l[w] = l;
  }
  __syncthreads();
  const float lt = s_l[0] + s_l[1] + s_l[2] + s_l[3];
  float o = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int s = gr + i * NG;
    const float f = s < a.nsplit ? s_f[s] : -1.0f;
    if (f >= 0.0f || f != f) o += f * x[i];  // a split without keys has no output
  }
  for (int s = gr + 8 * NG; s < a.nsplit; s += NG) {
    const float f = s_f[s];
    if (f >= 0.0f || f != f) o += f * po[(int64_t)s * D];
  }
  s_red[tid] = o;
  __syncthreads();
  if (gr == 0 && d < D) {
#pragma unroll
    for (int i = 1; i < NG; ++i) o += s_red[i * DT + d];
    static_cast<T*>(a.out)[row * D + d] = static_cast<T>(any ? o / lt : 0.0f);
    if (a.lse && d == 0) a.lse[row] = any ? Mt + (__log2f(lt) - WeightPlanes<T>::kBias) : -INFINITY;
  }
}

// ---------------------------------------------------------------- page selection
//
// One workgroup per (stream, key/value head): eight lanes a page, the scores'
// ordered 64-bit keys in LDS, then the num_selected largest (top_select.h): up to
// 256 pages one wave with the keys in registers (against the radix passes of the
// whole workgroup, pages scored alike: 9.9 and 11.0 us at 256 pages, 19.1 and
// 15.8 at 512), else those passes.  Latency: 6 MB of page sums (32 streams of 256 pages, 4
// heads of 64) would take 1.3 us, the kernel takes 6.9, and 38 for 4096 pages
// (134 MB, 3.6 TB/s).  Four pages a lane load at once without a branch, which took
// 11.0 to 6.9 us and 114 to 52 against a page at a time.

struct SelectArgs {
  const void* q;
  const float* sums;
  const int32_t* table;
  const int32_t* lengths;
  int32_t* out;
  int64_t num_pages;
  int32_t width, page, H, Hkv, G, D, S, first, local;
};

// Threads of a workgroup, by the table's width in pages (32 streams, 4 heads of
// 64, full tables): 512 against 1024 threads take 6.9 and 7.6 us at 256 pages,
// 9.8 and 10.4 at 512, 17.6 and 15.2 at 1024, 52 and 38 at 4096.
constexpr int kSelWide = 512;  // pages

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void page_select_kernel(SelectArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  uint64_t* keys = reinterpret_cast<uint64_t*>(lds);
  __shared__ double s_q[128];
  __shared__ ma_top::Scratch<THREADS> sc;
  const int tid = threadIdx.x;
  const int hk = blockIdx.x % (uint32_t)a.Hkv;
  const int64_t b = blockIdx.x / (uint32_t)a.Hkv;
  int64_t len = a.lengths[b];
  const int64_t cap = (int64_t)a.width * a.page;
  len = len < 0 ? 0 : (len > cap ? cap : len);
  const int n = (int)(((uint32_t)len + (uint32_t)a.page - 1) / (uint32_t)a.page);  // len <= cap < 2^31
  // the page slots of a group's pages load before the queries' sum, and a
  // group's sums before the products of the first
  constexpr int kRows = THREADS / 8, kGroup = 4;
  const int e = tid & 7, row = tid >> 3;
  int32_t ph[kGroup];
  auto slots = [&](int p0) {
#pragma unroll
    for (int g = 0; g < kGroup; ++g) {
      const int p = p0 + g * kRows + row;
      ph[g] = p < n ? a.table[b * a.width + p] : -1;
      if (ph[g] >= a.num_pages) ph[g] = -1;
    }
  };
  slots(0);
  if (tid < a.D) {
    const T* qp = static_cast<const T*>(a.q) + (b * a.H + (int64_t)hk * a.G) * a.D + tid;
    double s = 0.0;
    for (int i = 0; i < a.G; ++i) s += (double)(float)qp[(int64_t)i * a.D];
    s_q[tid] = s;
  }
  __syncthreads();
  const double ps = (double)a.page;
  // pages of a power of two: the product with 1 / page is the quotient (256
  // pages of 64 tokens 6.8 us, of 48 8.4; 4096 pages 38 and 61)
  const bool pow2 = (a.page & (a.page - 1)) == 0;
  const double inv = 1.0 / ps;
  const int dims = a.num_pages > 0 ? a.D : 0;
  for (int p0 = 0; p0 < n; p0 += kGroup * kRows) {
    if (p0) slots(p0);
    double s[kGroup] = {};
    for (int d = 4 * e; d < dims; d += 32) {
      float4 v[kGroup];
#pragma unroll
      for (int g = 0; g < kGroup; ++g) {
        const int64_t at = ph[g] < 0 ? 0 : ph[g];  // page 0's sums in place of none, unused
        v[g] = *reinterpret_cast<const float4*>(a.sums + (at * a.Hkv + hk) * a.D + d);
      }
      const double q0 = s_q[d], q1 = s_q[d + 1], q2 = s_q[d + 2], q3 = s_q[d + 3];
      if (pow2) {
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
          s[g] += (double)v[g].x * inv * q0;
          s[g] += (double)v[g].y * inv * q1;
          s[g] += (double)v[g].z * inv * q2;
          s[g] += (double)v[g].w * inv * q3;
        }
      } else {
#pragma unroll
        for (int g = 0; g < kGroup; ++g) {
          s[g] += (double)v[g].x / ps * q0;
          s[g] += (double)v[g].y / ps * q1;
          s[g] += (double)v[g].z / ps * q2;
          s[g] += (double)v[g].w / ps * q3;
        }
      }
    }
#pragma unroll
    for (int g = 0; g < kGroup; ++g) {
#pragma unroll
      for (int k = 1; k < 8; k <<= 1) s[g] += __shfl_xor(s[g], k, 64);
      const int p = p0 + g * kRows + row;
      if (e == 0 && p < n)
        keys[p] = ph[g] < 0 ? 0 : (p < a.first || p >= n - a.local ? ~0ull : ma_top::ordered(s[g]));
    }
  }
  __syncthreads();
  int32_t* out = a.out + (b * a.Hkv + hk) * (int64_t)a.S;
  if (n <= 256) {
    if (tid < 64) ma_top::wave_top<4>(keys, n, a.S, out);
  } else {
    ma_top::list_top<THREADS>(keys, n, a.S, out, sc);
  }
}

}  // namespace ma_paged
