// Element types of the operators that take bf16, fp16 and fp32: conversions, the
// matrix instructions of the 16-bit types and 16-byte row pieces. MFMA operands
// of both 16-bit types travel as bf16x8 bit patterns.
#pragma once

#include "common.hpp"

namespace solattn {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Two fp32 -> a packed fp16 pair, round to nearest even.
__device__ __forceinline__ uint32_t cvt_pk_f16(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) float f2;
  typedef __attribute__((ext_vector_type(2))) _Float16 h2;
  const f2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
}

struct Bf16 {
  using Raw = uint16_t;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return cvt_pk_bf16(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return lo_bf16(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return hi_bf16(w); }
  static __device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

struct Fp16 {
  using Raw = uint16_t;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return cvt_pk_f16(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w)));
  }
  static __device__ __forceinline__ float hi(uint32_t w) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w >> 16)));
  }
  static __device__ __forceinline__ f32x16 mfma32(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                  0, 0);
  }
};

struct Fp32 {
  using Raw = float;
};

// Eight consecutive values of a row (16-byte aligned) as fp32, and back with one rounding.
template <typename E>
struct Row8 {
  uint4 w;
  __device__ __forceinline__ void load(const typename E::Raw* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = E::lo(u[i]);
      x[2 * i + 1] = E::hi(u[i]);
    }
  }
  static __device__ __forceinline__ void store(typename E::Raw* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(x[4], x[5]),
                                              E::pack(x[6], x[7]));
  }
};
template <>
struct Row8<Fp32> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = reinterpret_cast<const float4*>(p)[0];
    b = reinterpret_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};

}  // namespace solattn
