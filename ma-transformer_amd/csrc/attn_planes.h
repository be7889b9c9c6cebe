// attn_planes.h -- float32 weights as operands of the 16-bit matrix cores.
#pragma once

#include "device_common.h"

namespace ma_dev {

// A float32 value enters a 16-bit product as a sum of 16-bit planes, so that
// nothing but the stored results is rounded to 16 bits.  bf16: three planes,
// each the rounding of what is left (24 bits, float32's exponent range).  f16
// has no bits below 2^-24, so its two planes (22 bits) hold the value times a
// power of two: kBias puts weights of at most 1 just below f16's maximum, and
// a sum keeps the bits of weights down to 2^-39 of its largest.
template <typename T>
struct WeightPlanes;

template <>
struct WeightPlanes<float> {
  static constexpr float kBias = 0.0f;
};

template <>
struct WeightPlanes<__bf16> {
  static constexpr int N = 3;
  static constexpr float kBias = 0.0f;
  uint4 w[N];
  // p0: elements 0..3, p1: elements 4..7 of the lane's eight contraction terms
  __device__ __forceinline__ void set(const float (&p0)[4], const float (&p1)[4]) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p0[i], x[4 + i] = p1[i];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[i] = Mma<__bf16>::pack2(x[2 * i], x[2 * i + 1]);
        if (k + 1 < N) {
          x[2 * i] -= __uint_as_float(q[i] << 16);
          x[2 * i + 1] -= __uint_as_float(q[i] & 0xffff0000u);
        }
      }
      w[k] = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
};

template <>
struct WeightPlanes<_Float16> {
  static constexpr int N = 2;
  static constexpr float kBias = 15.0f;
  uint4 w[N];
  __device__ __forceinline__ void set(const float (&p0)[4], const float (&p1)[4]) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = p0[i], x[4 + i] = p1[i];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q[i] = Mma<_Float16>::pack2(x[2 * i], x[2 * i + 1]);
        if (k + 1 < N) {
          const f16x2 h = __builtin_bit_cast(f16x2, q[i]);
          x[2 * i] -= (float)h[0];
          x[2 * i + 1] -= (float)h[1];
        }
      }
      w[k] = make_uint4(q[0], q[1], q[2], q[3]);
    }
  }
};

}  // namespace ma_dev
