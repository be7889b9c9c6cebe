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
//
// Op<T>: one MFMA operand's eight contraction terms of a lane (lane = 16 g + c
// holds terms 8 g .. 8 g + 7 of row, or column, c).  float32 takes eight
// 16x16x4 products for the one 16x16x32 of the 16-bit types.
template <typename T>
struct Op {
  using F = uint4;
  static __device__ __forceinline__ F zero() { return make_uint4(0, 0, 0, 0); }
  static __device__ __forceinline__ F load(const T* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ f32x4 mma(const F& a, const F& b, f32x4 c) { return Mma<T>::x32(a, b, c); }
  // any element infinite or NaN
  static __device__ __forceinline__ bool bad(const F& a) {
    constexpr uint32_t m = __is_same(T, __bf16) ? 0x7f80u : 0x7c00u, h = m << 16;
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    bool r = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) r = r || (w[i] & m) == m || (w[i] & h) == h;
    return r;
  }
};

struct F32x8 {
  float v[8];
};

template <>
struct Op<float> {
  using F = F32x8;
  static __device__ __forceinline__ F zero() { return F{{0, 0, 0, 0, 0, 0, 0, 0}}; }
  static __device__ __forceinline__ F load(const float* p) {
    F f;
    reinterpret_cast<float4*>(f.v)[0] = reinterpret_cast<const float4*>(p)[0];
    reinterpret_cast<float4*>(f.v)[1] = reinterpret_cast<const float4*>(p)[1];
    return f;
  }
  static __device__ __forceinline__ f32x4 mma(const F& a, const F& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = mfma_f32(a.v[i], b.v[i], c);
    return c;
  }
  static __device__ __forceinline__ bool bad(const F& a) {
    bool r = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) r = r || (__float_as_uint(a.v[i]) & 0x7f800000u) == 0x7f800000u;
    return r;
  }
};

// Reads a finished product into vector registers where it stands.  The wait
// states between an MFMA and the first vector instruction that reads its result
// are the compiler's to insert; hipcc (ROCm 7.2) left them out where the reader
// was the first instruction behind a branch that follows the MFMA, and the read
// returned the sum without its last product.  Results that are read behind a
// branch are settled before it.
__device__ __forceinline__ void settle(f32x4& x) { asm volatile("" : "+v"(x)); }

template <typename T>
struct WeightPlanes;

template <>
struct WeightPlanes<float> {
  static constexpr int N = 1;
  static constexpr float kBias = 0.0f;
  F32x8 w[N];
  __device__ __forceinline__ void set(const float (&p0)[4], const float (&p1)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[0].v[i] = p0[i], w[0].v[4 + i] = p1[i];
  }
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
