// top_select.h -- the indices of the S largest of n ordered keys, ascending,
// by one workgroup.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ma_top {

// Order-preserving 64-bit key of a score; NaN counts as -inf, -0 as 0.  Never
// 0 (which marks an entry that may not be listed) and below ~0 (always listed).
__device__ __forceinline__ uint64_t ordered(double x) {
  x = x != x ? -__builtin_inf() : x + 0.0;
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  return u >> 63 ? ~u : u | (1ull << 63);
}

template <int THREADS>
struct Scratch {
  uint32_t hist[256];
  uint32_t found[4];
  uint32_t wave[2][THREADS / 64];
};

// keys [n], n <= 64 R, in LDS; out [S].  Bisection from the top bit, by one wave
// with the keys in registers: a bit stays in the threshold where S keys reach
// it, and the search ends when exactly S do.  Equal keys go to the lowest
// indices.  Every lane of the wave calls it.
template <int R>
__device__ void wave_top(const uint64_t* keys, int n, int S, int32_t* out) {
  const int lane = threadIdx.x & 63;
  uint64_t k[R];
  int reach = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    k[r] = 64 * r + lane < n ? keys[64 * r + lane] : 0;
    reach += __popcll(__ballot(k[r] != 0));
  }
  uint64_t least = 1;  // `reach` keys are no smaller
  if (reach > S) {
    least = 0;
    for (int bit = 63; bit >= 0 && reach != S; --bit) {
      const uint64_t t = least | 1ull << bit;
      int c = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) c += __popcll(__ballot(k[r] >= t));
      if (c >= S) {
        least = t;
        reach = c;
      }
    }
  }
  // ascending output; of the keys at the threshold the first ones
  int above = 0;
  if (reach > S) {
#pragma unroll
    for (int r = 0; r < R; ++r) above += __popcll(__ballot(k[r] > least));
  }
  int ties = reach > S ? S - above : S, put = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const uint64_t below = (1ull << lane) - 1;
    const uint64_t e = __ballot(k[r] == least);
    const bool take = k[r] > least || (k[r] == least && (int)__popcll(e & below) < ties);
    ties -= (int)__popcll(e);
    const uint64_t b = __ballot(take);
    if (take) out[put + __popcll(b & below)] = 64 * r + lane;
    put += __popcll(b);
  }
  if (put + lane < S) out[put + lane] = -1;
}

// keys [n] in LDS; out [S].  Radix selection from the top byte: each pass
// counts the keys that share the prefix found so far by their next byte, and
// ends early when a bucket's end falls on S.  Equal keys go to the lowest
// indices.  Every thread of the workgroup calls it.
template <int THREADS>
__device__ void list_top(const uint64_t* keys, int n, int S, int32_t* out, Scratch<THREADS>& sc) {
  const int tid = threadIdx.x, lane = tid & 63;
  uint64_t prefix = 0, mask = 0;
  uint32_t need = (uint32_t)S;
  bool all = true;  // every key of the prefix's bucket is taken
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += THREADS) sc.hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t k = keys[i];
      if (k != 0 && (k & mask) == prefix) atomicAdd(&sc.hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid < 64) {
      // lane i holds the four buckets from the top: 255 - 4 i ...
      uint32_t h[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += h[i] = sc.hist[255 - 4 * lane - i];
      uint32_t inc = sum;
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) {
        const uint32_t y = __shfl_up(inc, k, 64);
        if (lane >= k) inc += y;
      }
      uint32_t before = inc - sum;
      if (lane == 63) sc.found[3] = inc;  // keys under this prefix
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < need && before + h[i] >= need) {
          sc.found[0] = (uint32_t)(255 - 4 * lane - i);
          sc.found[1] = before;
          sc.found[2] = h[i];
        }
        before += h[i];
      }
    }
    __syncthreads();
    if (sc.found[3] < need) break;  // only at the first byte: fewer keys than S, all taken
    const uint32_t bucket = sc.found[0], before = sc.found[1], size = sc.found[2];
    prefix |= (uint64_t)bucket << shift;
    mask |= 255ull << shift;
    need -= before;
    all = size == need;
    __syncthreads();  // found and hist have been read
    if (all) break;
  }
  __syncthreads();
  // ascending output: taken keys counted in index order; of the bucket's keys
  // the first `need`
  uint32_t put = 0, ties = 0;
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + tid;
    const uint64_t k = i < n ? keys[i] : 0;
    const bool tie = k != 0 && !all && (k & mask) == prefix;
    const uint64_t tb = __ballot(tie);
    if (lane == 0) sc.wave[0][tid >> 6] = (uint32_t)__popcll(tb);
    __syncthreads();
    uint32_t rank = ties + (uint32_t)__popcll(tb & ((1ull << lane) - 1)), tall = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
      const uint32_t x = sc.wave[0][w];
      if (w < (tid >> 6)) rank += x;
      tall += x;
    }
    ties += tall;
    const bool take = k != 0 && (tie ? rank < need : (k & mask) >= prefix);
    const uint64_t b = __ballot(take);
    if (lane == 0) sc.wave[1][tid >> 6] = (uint32_t)__popcll(b);
    __syncthreads();
    uint32_t pos = put + (uint32_t)__popcll(b & ((1ull << lane) - 1)), sum = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
      const uint32_t x = sc.wave[1][w];
      if (w < (tid >> 6)) pos += x;
      sum += x;
    }
    put += sum;
    if (take && pos < (uint32_t)S) out[pos] = i;
  }
  for (uint32_t j = put + tid; j < (uint32_t)S; j += THREADS) out[j] = -1;
}

}  // namespace ma_top
