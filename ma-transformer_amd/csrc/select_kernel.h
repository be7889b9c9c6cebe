// select_kernel.h -- the blocks whose mean key scores highest, per query.
#pragma once

#include "device_common.h"
#include "top_select.h"

namespace ma_select {

using namespace ma_dev;

typedef double f64x4 __attribute__((ext_vector_type(4)));

struct Args {
  const void* q;
  const void* k;
  double* mean;  // [B * Hkv][nbp][D]
  int32_t* out;
  int64_t N;
  int32_t units, H, Hkv, G, D, S, BS, nb, nbp, causal, first, local;  // units: B * Hkv; nbp: nb rounded up to 16
};

// Means of the blocks' keys, in float64: a sum of 16-bit keys is exact there,
// so equal blocks get equal means and a near tie falls the same way whoever
// computes it.
constexpr int kMeanThreads = 256;

template <typename T>
__global__ __launch_bounds__(kMeanThreads) void mean_kernel(Args a, int parts) {
  const int64_t x = blockIdx.x;
  const int part = (int)(x % parts);
  const int64_t bb = x / parts;
  const int blk = (int)(bb % a.nbp);
  const int64_t b = bb / a.nbp;
  const int e = part * kMeanThreads + threadIdx.x, row = a.Hkv * a.D;
  if (e >= row) return;
  const int64_t k0 = (int64_t)blk * a.BS;
  const int n = a.N - k0 < a.BS ? (a.N - k0 < 0 ? 0 : (int)(a.N - k0)) : a.BS;
  const T* p = static_cast<const T*>(a.k) + (b * a.N + k0) * row + e;
  double s = 0.0;
#pragma unroll 8
  for (int i = 0; i < n; ++i) s += (double)(float)p[(int64_t)i * row];
  const int h = e / a.D, d = e - h * a.D;
  a.mean[((b * a.Hkv + h) * a.nbp + blk) * a.D + d] = n ? s / (double)n : 0.0;
}

// Ordered 32-bit key of a score rounded to float32 (the rounding keeps the
// order, weakly); 0: may not be listed, ~0: always listed.
__device__ __forceinline__ uint32_t key32f(float x) {
  const int u = __float_as_int(x);
  return (uint32_t)u ^ ((uint32_t)(u >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t key32(double x) {
  const float f = (float)x;
  return key32f(f != f ? -INFINITY : f + 0.0f);
}
__device__ __forceinline__ float value32(uint32_t k) {
  return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// One wave lists the blocks of 16 queries.  float64 16x16x4 products of the
// means (rows) and the group's summed queries (columns) leave a query's scores
// in the four lanes of its column, 64 blocks a lane for a chunk of 256; the
// S-th largest is found by bisection over float32 keys in registers, sixteen
// queries at once.  Blocks that tie in float32 at the border are compared in
// float64 (a few queries in 10^5 on real scores; every one of a zero query).
// Sequences of more blocks go chunk by chunk with the S best carried over.
// 16384 queries of 8 heads of 64, 16 of 256 blocks of 64, bf16: 175 us, bound by
// vector instructions (12 bisection steps over up to 64 keys a lane); the
// products' floor at the card's float64 rate is 33.
constexpr int kRowWaves = 4;
constexpr int kChunkTiles = 16;
constexpr int kTies = 64 + 16 * kChunkTiles;

struct RowLds {
  double ts[kTies];
  double qs[128];
  int32_t idx[kTies];
  int32_t taken[kTies];
};

// dynamic LDS of a workgroup: per wave RowLds, then keys and blocks [16][S]
inline size_t row_lds_bytes(int S) { return kRowWaves * (sizeof(RowLds) + (size_t)16 * S * 8); }

template <typename T, int DP>
__global__ __launch_bounds__(64 * kRowWaves, 2) void rows_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  constexpr int SD = DP / 4;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
  uint8_t* base = lds + w * (sizeof(RowLds) + (size_t)16 * a.S * 8);
  RowLds* t = reinterpret_cast<RowLds*>(base);
  uint32_t* lk = reinterpret_cast<uint32_t*>(base + sizeof(RowLds));  // [16][S]
  int32_t* li = reinterpret_cast<int32_t*>(lk + 16 * a.S);
  const int64_t tiles = (a.N + 15) / 16;
  const int64_t id = (int64_t)blockIdx.x * kRowWaves + w;
  const int64_t unit = id / tiles, i0 = (id - unit * tiles) * 16;
  const int64_t b = unit / a.Hkv;
  const int hk = (int)(unit - b * a.Hkv), D = a.D, Q = D >> 2, S = a.S;
  if (unit >= a.units) return;  // the last workgroup's spare waves; there are no barriers
  const int64_t i = i0 + c < a.N ? i0 + c : a.N - 1;
  const int own = (int)(i / a.BS);

  double qs[SD];
  const T* qp = static_cast<const T*>(a.q) + ((b * a.N + i) * a.H + (int64_t)hk * a.G) * D + g * Q;
#pragma unroll
  for (int s = 0; s < SD; ++s) qs[s] = 0.0;
  for (int h = 0; h < a.G; ++h)
#pragma unroll
    for (int s = 0; s < SD; ++s)
      if (s < Q) qs[s] += (double)(float)qp[(int64_t)h * D + s];

  const double* mp = a.mean + unit * a.nbp * D;
  const int64_t ilast = i0 + 15 < a.N ? i0 + 15 : a.N - 1;
  const int nt = a.causal ? (int)(ilast / a.BS) / 16 + 1 : a.nbp / 16;
  int have = 0;  // listed so far (carried)
  const int own_first = (int)(i0 / a.BS);  // the first query's block: no query's is lower
  for (int t0 = 0; t0 < nt; t0 += kChunkTiles) {
    uint32_t key[kChunkTiles][4];
    // the next tile's means are loaded while this one's are multiplied, where the
    // registers hold both (185 -> 176 us at head_dim 64)
    constexpr bool kAhead = DP <= 64;
    double2 x[SD / 2];
    auto means = [&](int t) {
      const double* row = mp + (int64_t)(16 * t + c) * D + g * Q;
#pragma unroll
      for (int s = 0; s < SD / 2; ++s) {
        x[s] = make_double2(0.0, 0.0);
        if (2 * s < Q) x[s] = *reinterpret_cast<const double2*>(row + 2 * s);
      }
    };
    if (kAhead) means(t0);
#pragma unroll
    for (int u = 0; u < kChunkTiles; ++u) {
#pragma unroll
      for (int r = 0; r < 4; ++r) key[u][r] = 0;
      if (t0 + u < nt) {
        f64x4 acc = {0, 0, 0, 0}, acc2 = {0, 0, 0, 0};
        if (!kAhead) means(t0 + u);
        double2 y[SD / 2];
#pragma unroll
        for (int s = 0; s < SD / 2; ++s) y[s] = x[s];
        if (kAhead && t0 + u + 1 < nt) means(t0 + u + 1);
#pragma unroll
        for (int s = 0; s < SD / 2; ++s) {
          acc = __builtin_amdgcn_mfma_f64_16x16x4f64(y[s].x, qs[2 * s], acc, 0, 0, 0);
          acc2 = __builtin_amdgcn_mfma_f64_16x16x4f64(y[s].y, qs[2 * s + 1], acc2, 0, 0, 0);
        }
        acc += acc2;
#pragma unroll
        for (int r = 0; r < 4; ++r) key[u][r] = key32(acc[r]);
        const int b0 = 16 * (t0 + u);
        if (b0 < a.first || b0 + 15 > own_first - a.local) {  // not every block is an ordinary candidate
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int blk = b0 + 4 * r + g;  // float64 results: row 4 r + g
            const bool cand = blk < a.nb && (!a.causal || blk <= own);
            const bool forced = blk < a.first || (blk <= own && blk > own - a.local);
            key[u][r] = cand ? (forced ? ~0u : key[u][r]) : 0u;
          }
        }
      }
    }
    // carried blocks, in the query's list: slot 4 r + g
    const bool carried = t0 > 0;
    auto ckey = [&](int r) { return 4 * r + g < have ? lk[c * S + 4 * r + g] : 0u; };
    auto cblk = [&](int r) { return 4 * r + g < have ? li[c * S + 4 * r + g] : 0; };
    const int cr = (S + 3) >> 2;
    auto sum4 = [&](int x) {
      x += __shfl_xor(x, 16, 64);
      return x + __shfl_xor(x, 32, 64);
    };
    auto at_least = [&](uint32_t th) {
      int n = 0;
#pragma unroll
      for (int q = 0; q < kChunkTiles; q += 4)
        if (t0 + q < nt)  // four tiles at a time, as far as there are any
#pragma unroll
          for (int u = q; u < q + 4; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) n += key[u][r] >= th;
      if (carried)
        for (int r = 0; r < cr; ++r) n += ckey(r) >= th;
      return sum4(n);
    };
    // the largest threshold that at least S keys reach
    uint32_t mx = 0, mn = ~0u;
    auto see = [&](uint32_t k) {
      mx = k != ~0u && k > mx ? k : mx;
      mn = k != 0 && k < mn ? k : mn;
    };
#pragma unroll
    for (int q = 0; q < kChunkTiles; q += 4)
      if (t0 + q < nt)
#pragma unroll
        for (int u = q; u < q + 4; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) see(key[u][r]);
    if (carried)
      for (int r = 0; r < cr; ++r) see(ckey(r));
    for (int k = 16; k < 64; k <<= 1) {
      const uint32_t x = __shfl_xor(mx, k, 64), y = __shfl_xor(mn, k, 64);
      mx = x > mx ? x : mx;
      mn = y < mn ? y : mn;
    }
    const int total = at_least(1u), forced = at_least(~0u);
    uint32_t thr = 1u, lo = mn, hi = mx + 1;
    int flo = total;  // keys at or above lo
    bool done = total <= S, tie = false;
    if (!done && forced >= S) {
      thr = ~0u;
      done = true;
    }
    for (int step = 0; __ballot(!done); ++step) {
      uint32_t mid = lo + ((hi - lo) >> 1);
      const float fl = value32(lo), fh = value32(hi);
      // halving the values converges in about 12 steps on ordinary scores; from
      // the 16th on the keys are halved, which ends in 32
      if (step < 16 && fabsf(fl) < 1e30f && fabsf(fh) < 1e30f) mid = key32f(0.5f * (fl + fh) + 0.0f);
      mid = mid <= lo ? lo + 1 : (mid >= hi ? hi - 1 : mid);
      if (!done && hi - lo <= 1) {
        thr = lo;
        tie = flo > S;
        done = true;
      }
      const int n = at_least(mid);
      if (!done) {
        if (n == S) {
          thr = mid;
          done = true;
        } else if (n > S) {
          lo = mid;
          flo = n;
        } else {
          hi = mid;
        }
      }
    }
    // float32 ties at the border, one query at a time
    uint64_t todo = __ballot(tie && g == 0);
    while (todo) {
      const int qx = __builtin_ctzll(todo);
      todo &= todo - 1;
      const uint32_t th = (uint32_t)__builtin_amdgcn_readlane((int)thr, qx);
      int m = 0;
      const int need = S - __builtin_amdgcn_readlane(at_least(th + 1), qx);
      auto collect = [&](uint32_t k, int32_t blk) {
        const uint64_t bal = __ballot(c == qx && k == th);
        if (c == qx && k == th) t->idx[m + __popcll(bal & ((1ull << lane) - 1))] = blk;
        m += __popcll(bal);
      };
      if (carried)
        for (int r = 0; r < cr; ++r) collect(ckey(r), cblk(r));
#pragma unroll
      for (int u = 0; u < kChunkTiles; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) collect(key[u][r], 16 * (t0 + u) + 4 * r + g);
      const T* qr = static_cast<const T*>(a.q) +
                    ((b * a.N + (i0 + qx < a.N ? i0 + qx : a.N - 1)) * a.H + (int64_t)hk * a.G) * D;
      for (int d = lane; d < D; d += 64) {
        double s = 0.0;
        for (int h = 0; h < a.G; ++h) s += (double)(float)qr[(int64_t)h * D + d];
        t->qs[d] = s;
      }
      wave_fence();
      for (int e = lane; e < m; e += 64) {
        const double* row = mp + (int64_t)t->idx[e] * D;
        double s = 0.0;
        for (int d = 0; d < D; ++d) s += row[d] * t->qs[d];
        t->ts[e] = s;
        t->taken[e] = 0;
      }
      wave_fence();
      for (int k = 0; k < need; ++k) {
        uint64_t best = 0;
        int at = kTies;
        for (int e = lane; e < m; e += 64) {
          const uint64_t o = t->taken[e] ? 0 : ma_top::ordered(t->ts[e]);
          if (o > best) best = o, at = e;
        }
#pragma unroll
        for (int x = 32; x >= 1; x >>= 1) {
          const uint64_t ob = (uint64_t)__shfl_xor((long long)best, x, 64);
          const int oa = __shfl_xor(at, x, 64);
          if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
        }
        if (lane == 0 && at < kTies) t->taken[at] = 1;
        wave_fence();
      }
      m = 0;
      auto drop = [&](uint32_t& k) {
        const uint64_t bal = __ballot(c == qx && k == th);
        if (c == qx && k == th && !t->taken[m + __popcll(bal & ((1ull << lane) - 1))]) k = 0;
        m += __popcll(bal);
      };
      if (carried)
        for (int r = 0; r < cr; ++r) {
          uint32_t k = ckey(r);
          drop(k);
          if (4 * r + g < have) lk[c * S + 4 * r + g] = k;
        }
#pragma unroll
      for (int u = 0; u < kChunkTiles; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) drop(key[u][r]);
      wave_fence();
    }
    // the listed ones in ascending order: carried ones come first
    int put = 0;
    auto keep = [&](uint32_t k, int32_t blk) {
      const uint64_t bal = __ballot(k >= thr);
      if (!bal) return;
      const uint32_t four = (uint32_t)(bal >> c & 1) | (uint32_t)(bal >> (c + 16) & 1) << 1 |
                            (uint32_t)(bal >> (c + 32) & 1) << 2 | (uint32_t)(bal >> (c + 48) & 1) << 3;
      if (k >= thr) {
        const int at = put + __popc(four & ((1u << g) - 1));
        if (at < S) lk[c * S + at] = k, li[c * S + at] = blk;
      }
      put += __popc(four);
    };
    wave_fence();
    if (carried)
      for (int r = 0; r < cr; ++r) {  // in place: nothing moves up
        const uint32_t k = ckey(r);
        const int32_t blk = cblk(r);
        wave_fence();
        keep(k, blk);
        wave_fence();
      }
#pragma unroll
    for (int q = 0; q < kChunkTiles; q += 4)
      if (t0 + q < nt)
#pragma unroll
        for (int u = q; u < q + 4; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) keep(key[u][r], 16 * (t0 + u) + 4 * r + g);
    have = put < S ? put : S;
    wave_fence();
  }
  int32_t* out = a.out + (b * a.N * a.Hkv + hk) * S;
  for (int e = lane; e < 16 * S; e += 64) {
    const int x = e / S, j = e - x * S;
    const int n = __shfl(have, x, 64);
    if (i0 + x < a.N) out[(i0 + x) * a.Hkv * S + j] = j < n ? li[x * S + j] : -1;
  }
}

}  // namespace ma_select
