// What prompt attention (64 keys a step) and attention over keys that sequences share (32 a step)
// have in common: the layout of a step's K and V in LDS, its reads, and the constants of the lazily
// moved reference maximum.
#pragma once

#include "common.h"

namespace rspx {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kKeys = 64;            // keys of a step of prompt attention; shared keys come in multiples of it
constexpr float kTau = 8.0f;         // log2 headroom before the reference maximum moves
constexpr float kNone = -1e30f;      // reference maximum before the first key

__device__ __forceinline__ s16x4 tr_read(const lds_char* __restrict__ p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
}

// c + both bf16 of x, rounded to nearest (measured: 63 of 64 sums as one rounding, none by more
// than 0.52 of a step).
__device__ __forceinline__ float dot2(uint32_t x, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x), __builtin_bit_cast(bf16x2, 0x3f803f80u), c, false);
}
// LDS reads of what is in place (its loads waited for, the barrier passed).  __restrict__:
// without alias information the compiler waits for every load to LDS in flight, the next
// steps' included, ahead of the first read.
__device__ __forceinline__ u32x4 read16(const lds_char* __restrict__ p) {
  return *(const __attribute__((address_space(3))) u32x4*)p;
}

// A barrier that does not wait for the loads in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// 16-byte unit swizzles of a staged row of U units, 256 bytes of banks: sixteen consecutive
// keys' units of one column lie in different banks (K); so do four keys' four units, and
// eight keys' two (V).
template <int D>
__device__ __forceinline__ int kswizzle(int key) {
  constexpr int U = D / 8;
  if constexpr (U >= 16) return key % 16;
  else return (key / (16 / U)) % U;
}
template <int D>
__device__ __forceinline__ int vswizzle(int key) {
  constexpr int U = D / 8;
  const int odd = 2 * ((key >> 2) & 1);
  if constexpr (U >= 16) return 4 * (key % 4) + odd;
  else if constexpr (U == 8) return 4 * ((key >> 1) & 1) + odd;
  else return odd;
}

}  // namespace rspx
