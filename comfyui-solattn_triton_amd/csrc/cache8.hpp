// The 8-bit rows of a key-value cache: codes of D channels and one exponent byte b, a
// value is code 2^(b - 127). A power of two costs int8 up to a bit of its seven, and
// e4m3 nothing; what it buys is that a cached value is a 16-bit number exactly, so every
// kernel that reads the cache computes with the same values as one that reads them back.
//
// Of a row with largest magnitude a, 2^(b - 127) is the smallest power of two with
// a <= 127 2^(b - 127) (int8) or 448 2^(b - 127) (e4m3); codes are rounded to nearest
// even, from 32 bits: by half a step at most, 2^(b - 128) of int8, 2^-4 of a value of e4m3
// (2^(b - 137) below its smallest normal). Rows below 2^-110 are zeros (b = 0, codes 0).
// A row with a NaN or an infinity reads as NaN: b = 255 (the bits of an infinity) and codes
// 0 (int8) or NaN (e4m3).
#pragma once

#include "elem.hpp"

namespace solattn {

constexpr uint32_t kTinyRow = (127u - 110u) << 23;  // bits of 2^-110
constexpr uint32_t kInfBits = 0x7F800000u;

__device__ __forceinline__ float power_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// The power of byte i of a word, in one instruction (an AND and a shift where the compiler chooses).
__device__ __forceinline__ float power_at(uint32_t word, int i) {
  uint32_t x;
#define SOLATTN_BYTE_SHL(sel) \
  asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:" sel : "=v"(x) : "v"(23), "v"(word))
  if (i == 0)
    SOLATTN_BYTE_SHL("BYTE_0");
  else if (i == 1)
    SOLATTN_BYTE_SHL("BYTE_1");
  else if (i == 2)
    SOLATTN_BYTE_SHL("BYTE_2");
  else
    SOLATTN_BYTE_SHL("BYTE_3");
#undef SOLATTN_BYTE_SHL
  return __uint_as_float(x);
}

// Exponent byte of a row whose largest magnitude has the bits `top`; unit: what the factor
// of the codes (2^-that) is multiplied with them as.
__device__ __forceinline__ uint32_t row_exponent(uint32_t top, uint32_t past, int shift, float& unit) {
  // a mantissa above that of 127 = 1.984375 2^6 (448 = 1.75 2^8) takes the next power
  const uint32_t e = (top + past) >> 23;
  const bool none = top < kTinyRow, bad = top >= kInfBits;
  const uint32_t b = e - shift;
  unit = none || bad ? 0.f : __uint_as_float((254u - b) << 23);
  return bad ? 255u : none ? 0u : b;
}

// The largest over the LPR lanes of a row.
template <int LPR>
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
#define SOLATTN_DPP_MAX(ctrl) \
  x = max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), ctrl, 0xf, 0xf, false)))
  SOLATTN_DPP_MAX(0xB1);   // quad_perm 1 0 3 2
  SOLATTN_DPP_MAX(0x4E);   // quad_perm 2 3 0 1
  SOLATTN_DPP_MAX(0x141);  // row_half_mirror
  if constexpr (LPR == 16) SOLATTN_DPP_MAX(0x140);  // row_mirror
#undef SOLATTN_DPP_MAX
  return x;
}

// A cache of codes [pages, page, Hkv, D] and exponents [pages, Hkv, page]; strides in bytes.
struct CodePages {
  uint8_t* codes;
  int64_t p, s, h;
  uint8_t* exps;
  int64_t ep, eh;
};

// A row of fp32 values, eight a lane, to its place in the cache (every lane of a wave comes
// here; active: the lane holds channels, on: the row has a place).
template <typename C, int LPR>
__device__ __forceinline__ void put_codes(const float (&x)[8], const CodePages& to, int64_t page, int64_t slot, int h,
                                          int l, bool active, bool on) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  top = row_max<LPR>(active ? top : 0u);
  float unit;
  const uint32_t b = row_exponent(top, C::kPast, C::kShift, unit);
  if (!on) return;
  if (active) *reinterpret_cast<uint2*>(to.codes + page * to.p + slot * to.s + h * to.h + 8 * l) = C::encode(x, unit, b == 255u);
  if (l == 0) to.exps[page * to.ep + h * to.eh + slot] = static_cast<uint8_t>(b);
}

struct Int8Codes {
  static constexpr uint32_t kPast = 0x01FFFFu;  // 0x800000 - 0x7E0000 - 1
  static constexpr int kShift = 6;
  static constexpr uint32_t kFp16Byte = 127 + 8;  // fp16 holds 128 2^8, not 128 2^9
  // Eight values times the row's unit as codes; bad: the row holds a NaN or an infinity.
  static __device__ __forceinline__ uint2 encode(const float (&x)[8], float unit, bool bad) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        c[i] = static_cast<uint32_t>(static_cast<int>(__builtin_rintf(bad ? 0.f : x[4 * h + i] * unit)));
      const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
      w[h] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    }
    return make_uint2(w[0], w[1]);
  }
  static __device__ __forceinline__ float value(uint32_t w, int i) {
    return static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  }
  // Codes i and i + 1 (i even) of a word as a packed pair of E.
  template <typename E>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, int i) {
    return E::pack(value(w, i), value(w, i + 1));
  }
  // Code i of two words as a packed bf16 pair.
  static __device__ __forceinline__ uint32_t across(uint32_t w0, uint32_t w1, int i) {
    return cvt_pk_bf16(value(w0, i), value(w1, i));
  }
  // Codes i and i + 1 times the row's power as a packed pair of E.
  template <typename E>
  static __device__ __forceinline__ uint32_t scaled(uint32_t w, int i, float power) {
    return E::pack(value(w, i) * power, value(w, i + 1) * power);
  }
};

struct Fp8Codes {
  static constexpr uint32_t kPast = 0x1FFFFFu;  // 0x800000 - 0x600000 - 1
  static constexpr int kShift = 8;
  static constexpr uint32_t kFp16Byte = 127 + 7;  // fp16 holds 448 2^7, not 448 2^8
  static __device__ __forceinline__ uint2 encode(const float (&x)[8], float unit, bool bad) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] * unit, x[4 * h + 1] * unit, 0, false);
      w[h] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] * unit, x[4 * h + 3] * unit, lo, true));
      if (unit == 0.f) w[h] = bad ? 0x7F7F7F7Fu : 0u;  // (a row of zeros: without the signs that -x * 0 has)
    }
    return make_uint2(w[0], w[1]);
  }
  template <typename E>
  static __device__ __forceinline__ uint32_t scaled(uint32_t w, int i, float power) {
    if constexpr (__is_same(E, Bf16)) {
      return i ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, true))
               : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, false));
    } else {
      return i ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, true))
               : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, power, false));
    }
  }
  template <typename E>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, int i) {
    return scaled<E>(w, i, 1.f);
  }
  static __device__ __forceinline__ uint32_t across(uint32_t w0, uint32_t w1, int i) {
    // (the codes of two channels side by side: their two conversions share the permute)
    return scaled<Bf16>(__builtin_amdgcn_perm(w1, w0, i & 2 ? 0x07030602u : 0x05010400u), i & 1 ? 2 : 0, 1.f);
  }
};

}  // namespace solattn
