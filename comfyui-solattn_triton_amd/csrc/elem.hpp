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
  // The instructions of a hand-ordered stream (fwd_common.hpp has the rules that its
  // writer keeps): MFMAs, and p = exp2(s c + neg) of two scores, rounded, packed and
  // added to the row sum as rounded.
  static __device__ __forceinline__ void amfma0(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ void amfma(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ void amfma_first(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("s_nop 2\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
  }
  // (two wait states in front: b may have been written by the VALU just before)
  static __device__ __forceinline__ void amfma_after_valu(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ void amfma_tie(f32x16& d, const bf16x8& a, const bf16x8& b, f32x16& s) {
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %2, %3, %0\n\ts_nop 3" : "+v"(d), "+v"(s) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ uint32_t exp_pair(float s0, float s1, float c, float neg, float& sum) {
    uint32_t p;
    float t0, t1;
    asm volatile(
        "v_fma_f32 %2, %4, %6, %7\n\t"
        "v_fma_f32 %3, %5, %6, %7\n\t"
        "v_exp_f32 %2, %2\n\t"
        "v_exp_f32 %3, %3\n\t"
        "s_nop 0\n\t"
        "v_cvt_pk_bf16_f32 %0, %2, %3\n\t"
        "v_dot2_f32_bf16 %1, %0, %8, %1"
        : "=&v"(p), "+v"(sum), "=&v"(t0), "=&v"(t1)
        : "v"(s0), "v"(s1), "v"(c), "v"(neg), "s"(0x3F803F80u));
    return p;
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
  // The instructions of a hand-ordered stream (fwd_common.hpp has the rules that its
  // writer keeps): MFMAs, and p = exp2(s c + neg) of two scores, rounded, packed and
  // added to the row sum as rounded.
  static __device__ __forceinline__ void amfma0(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ void amfma(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ void amfma_first(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("s_nop 2\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
  }
  // (two wait states in front: b may have been written by the VALU just before)
  static __device__ __forceinline__ void amfma_after_valu(f32x16& d, const bf16x8& a, const bf16x8& b) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ void amfma_tie(f32x16& d, const bf16x8& a, const bf16x8& b, f32x16& s) {
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %2, %3, %0\n\ts_nop 3" : "+v"(d), "+v"(s) : "v"(a), "v"(b));
  }
  static __device__ __forceinline__ uint32_t exp_pair(float s0, float s1, float c, float neg, float& sum) {
    uint32_t p;
    float t0, t1;
    asm volatile(
        "v_fma_f32 %2, %4, %6, %7\n\t"
        "v_fma_f32 %3, %5, %6, %7\n\t"
        "v_exp_f32 %2, %2\n\t"
        "v_exp_f32 %3, %3\n\t"
        "s_nop 0\n\t"
        "v_cvt_pk_f16_f32 %0, %2, %3\n\t"
        "v_dot2_f32_f16 %1, %0, %8, %1"
        : "=&v"(p), "+v"(sum), "=&v"(t0), "=&v"(t1)
        : "v"(s0), "v"(s1), "v"(c), "v"(neg), "s"(0x3C003C00u));
    return p;
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

// Asks for every 64-byte line of a kernel's arguments at once: left to their first uses,
// they come one after the other, each a round trip to memory that the host has just written.
template <typename A>
__device__ __forceinline__ void fetch_arguments(const A& a) {
  constexpr int N = sizeof(A) / 4;
  uint32_t w[N];
  __builtin_memcpy(w, &a, N * 4);
#pragma unroll
  for (int i = 0; i < N; i += 16) asm volatile("" ::"s"(w[i]));
}

// Division by a number that the host knows: exact for n < 2^31 (mul = ceil(2^(31 + log2)
// / d), an error below 2^-31 n; mul 0: a power of two).
struct Divisor {
  uint32_t d, mul, shift;
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return mul ? __umulhi(n, mul) >> shift : n >> shift; }
  __device__ __forceinline__ uint32_t split(uint32_t& n) const {  // n becomes n / d; returns the remainder
    const uint32_t q = of(n), r = n - q * d;
    n = q;
    return r;
  }
};
inline Divisor divisor(int64_t d) {
  uint32_t log2 = 0;
  while ((1ll << log2) < d) ++log2;
  if ((1ll << log2) == d) return {static_cast<uint32_t>(d), 0, log2};
  return {static_cast<uint32_t>(d), static_cast<uint32_t>(((1ull << (31 + log2)) + d - 1) / d), log2 - 1};
}

}  // namespace solattn
