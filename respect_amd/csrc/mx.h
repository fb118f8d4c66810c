// Rows of a KV cache in bf16 or in the microscaled formats of 8 and 4 bits, for gfx950.
//
// BITS names the format: 16 bf16, 8 e4m3 codes, 4 e2m1 codes (the first of two in the low
// half of a byte).  32 consecutive codes share a scale byte e, 2^(e - 127).  Every value is
// exact in bf16: at most 4 significant bits, exponents of -126 and up (a scale is 2^-117 or
// more); but 2^128, to which numbers next to bf16's largest round, is an infinity there.  The converters take the scale as a float of which they use the exponent alone, so
// e << 23 is it; 255, which marks a group that held an infinity or a NaN, reads as NaN.  (All
// bf16 inputs and all codes at nine scales: equal to the definition, bit for bit.)
#pragma once

#include "common.h"

namespace rspx {

constexpr int kGroup = 32;           // elements of a scale
constexpr int kLeastScale = 10;      // 2^-117: e4m3's smallest code then stands for 2^-126

__device__ __forceinline__ float mx_scale(uint32_t e) { return __uint_as_float(e << 23); }

// The scales of up to 128 elements as a word, the first ones in its low byte; any alignment.
template <int D>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* p) {
  if constexpr (D >= 128) {
    uint32_t w;
    __builtin_memcpy(&w, p, 4);
    return w;
  } else if constexpr (D == 64) {
    uint16_t w;
    __builtin_memcpy(&w, p, 2);
    return w;
  } else {
    return *p;
  }
}
// Scale i of a row, from the word that holds it.
__device__ __forceinline__ float scale_in(uint32_t w, int i) { return mx_scale(__builtin_amdgcn_ubfe(w, 8 * (i & 3), 8)); }

typedef short s16x2 __attribute__((ext_vector_type(2)));

// Non-template wrappers: the host pass rejects these builtins inside templates.
__device__ __forceinline__ u32x4 values_of_fp8(uint32_t a, uint32_t b, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))};
}
__device__ __forceinline__ u32x4 values_of_fp4(uint32_t a, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(a, scale, 3))};
}
// Codes of four bf16 values (two words) in e4m3, of eight in e2m1.  (By value: a bit cast of an
// element of a vector in memory reads the vector's first.)
__device__ __forceinline__ uint32_t fp8_of(uint32_t a, uint32_t b, float scale) {
  s16x2 w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, a), scale, false);
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(w, __builtin_bit_cast(bf16x2, b), scale, true));
}
__device__ __forceinline__ uint32_t fp4_of(uint32_t x0, uint32_t x1, uint32_t x2, uint32_t x3, float scale) {
  uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf16x2, x0), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, x1), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, x2), scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, x3), scale, 3);
}

// W bytes of memory as W / 4 words; the address is W-byte aligned.
template <int W>
struct Words {
  uint32_t x[W / 4];
};
template <int W>
__device__ __forceinline__ Words<W> load_words(const char* p) {
  Words<W> r;
  if constexpr (W == 16) {
    const u32x4 y = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.x[i] = y[i];
  } else if constexpr (W == 8) {
    const u32x2 y = *reinterpret_cast<const u32x2*>(p);
    r.x[0] = y[0], r.x[1] = y[1];
  } else {
    r.x[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return r;
}

// Elements 8 i .. 8 i + 7 of W bytes of a row as bf16.
template <int BITS, int W>
__device__ __forceinline__ u32x4 eight(const Words<W>& r, int i, float scale) {
  if constexpr (BITS == 16) return u32x4{r.x[4 * i], r.x[4 * i + 1], r.x[4 * i + 2], r.x[4 * i + 3]};
  else if constexpr (BITS == 8) return values_of_fp8(r.x[2 * i], r.x[2 * i + 1], scale);
  else return values_of_fp4(r.x[i], scale);
}

}  // namespace rspx
