// Rows of a paged KV cache written in the microscaled formats, and rows of any format read
// back as bf16, for gfx950 (mx.h has the formats).
//
//   rspx_kv_write_mx  per head and 32 elements x of a row: s the smallest integer with
//                     max |x| <= M 2^s (M the largest code: 448, 6) and s >= -117;
//                     codes rne(x 2^-s), scale byte s + 127
//   rspx_kv_read      the values that the codes of given rows stand for, exact in bf16
//
// A thread takes eight elements of K and of V, so four neighbours hold a group and find its
// maximum by two exchanges; |x| of bf16 compares as an integer, and s comes of the
// maximum's own bits: its exponent, one more where its mantissa passes M's.  A workgroup takes
// consecutive rows of one head, which lie together in the pool where the slots follow one
// another: by token and head instead, the lines of a pool would be written in parts by
// different L2s.  What bounds both is the bytes of the rows.
#include <algorithm>

#include "mx.h"
#include "respect_amd.h"

namespace rspx {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kBlocksPerLaunch = 1 << 23;   // a grid dimension holds 2^32 threads

struct Rows {
  char *codes, *scales;
  int64_t ch, cn, sh, sn;              // head and slot strides in bytes
};
struct Tokens {
  uint16_t* x;
  int64_t st, sh;
};

// The largest of x over the four lanes of a group.
__device__ __forceinline__ uint32_t max_of_group(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xf, 0xf, true));   // lanes 1 0 3 2
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xf, 0xf, true));  // lanes 2 3 0 1
}

template <int BITS>
__device__ __forceinline__ void quantise(const u32x4& x, char* codes, char* scale, bool first) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i] & 0x7fff7fffu));
  const uint32_t top = max_of_group(max((uint32_t)m[0], (uint32_t)m[1]));
  // top's exponent, raised by a mantissa past 1.75 (448 = 1.75 2^8) or 1.5 (6 = 1.5 2^2).
  const int e = max((int)((top + (BITS == 8 ? 0x1f : 0x3f)) >> 7) - (BITS == 8 ? 8 : 2), kLeastScale);
  const bool none = top >= 0x7f80;     // an infinity or a NaN
  const float s = mx_scale(e);
  if constexpr (BITS == 8) {
    const u32x2 c = {fp8_of(x[0], x[1], s), fp8_of(x[2], x[3], s)};
    *reinterpret_cast<u32x2*>(codes) = none ? u32x2{0, 0} : c;
  } else {
    const uint32_t c = fp4_of(x[0], x[1], x[2], x[3], s);
    *reinterpret_cast<uint32_t*>(codes) = none ? 0 : c;
  }
  if (first) *reinterpret_cast<uint8_t*>(scale) = (uint8_t)(none ? 255 : e);
}

// Workgroup (rows, head): `per` rows of U = D / 8 threads each.
template <int BITS>
__global__ __launch_bounds__(kThreads) void kv_write_mx_kernel(Tokens k, Tokens v, const int* slots, int T, int cap, Rows ck,
                                                               Rows cv, int U, int per, int64_t first) {
  const int r = threadIdx.x / U, c = threadIdx.x - r * U, h = blockIdx.y;
  const int64_t t = first + (int64_t)blockIdx.x * per + r;
  if (r >= per || t >= T) return;      // whole groups: U is a multiple of four
  const u32x4 a = *reinterpret_cast<const u32x4*>(k.x + t * k.st + h * k.sh + 8 * c);
  const u32x4 b = *reinterpret_cast<const u32x4*>(v.x + t * v.st + h * v.sh + 8 * c);
  const int slot = slots[t];
  if (slot < 0 || slot >= cap) return;
  const bool lead = c % 4 == 0;
  quantise<BITS>(a, ck.codes + h * ck.ch + slot * ck.cn + c * BITS, ck.scales + h * ck.sh + slot * ck.sn + c / 4, lead);
  quantise<BITS>(b, cv.codes + h * cv.ch + slot * cv.cn + c * BITS, cv.scales + h * cv.sh + slot * cv.sn + c / 4, lead);
}

template <int BITS>
__device__ __forceinline__ u32x4 read_eight(const Rows& p, int h, int slot, int c) {
  float s = 0.f;
  if constexpr (BITS < 16) s = mx_scale(*reinterpret_cast<const uint8_t*>(p.scales + h * p.sh + slot * p.sn + c / 4));
  return eight<BITS>(load_words<BITS>(p.codes + h * p.ch + slot * p.cn + c * BITS), 0, s);
}

template <int BITS>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(Rows ck, Rows cv, const int* slots, int T, int cap, Tokens k,
                                                           Tokens v, int U, int per, int64_t first) {
  const int r = threadIdx.x / U, c = threadIdx.x - r * U, h = blockIdx.y;
  const int64_t t = first + (int64_t)blockIdx.x * per + r;
  if (r >= per || t >= T) return;
  const int slot = slots[t];
  u32x4 a, b;
  if (slot >= 0 && slot < cap) {
    a = read_eight<BITS>(ck, h, slot, c);
    b = read_eight<BITS>(cv, h, slot, c);
  } else {
    a = b = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  }
  *reinterpret_cast<u32x4*>(k.x + t * k.st + h * k.sh + 8 * c) = a;
  *reinterpret_cast<u32x4*>(v.x + t * v.st + h * v.sh + 8 * c) = b;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What both calls check of the pools; strides come in the pool's elements.
int rows_ok(const Rows& p, int D, int bits) {
  if (!p.codes || (bits < 16 && !p.scales)) return RSPX_EINVAL;
  if (p.cn < (int64_t)D * bits / 8 || p.ch < 0 || (bits < 16 && (p.sn < D / kGroup || p.sh < 0))) return RSPX_EINVAL;
  return !al16(p.codes) || p.ch % 16 || p.cn % 16 ? RSPX_EALIGN : RSPX_OK;
}

int sizes_ok(int T, int cap, int HK, int D, int bits) {
  if (T < 0 || cap < 0 || HK < 1 || D < 1) return RSPX_EINVAL;
  if (bits != 16 && bits != 8 && bits != 4) return RSPX_EUNSUPPORTED;
  if (D % (bits == 16 ? 8 : kGroup) || D > 8 * kThreads || HK > 65535) return RSPX_EUNSUPPORTED;
  return RSPX_OK;
}

int tokens_ok(const Tokens& t) {
  if (!t.x) return RSPX_EINVAL;
  return !al16(t.x) || t.st % 8 || t.sh % 8 ? RSPX_EALIGN : RSPX_OK;
}

template <class F>
int by_rows(int T, int D, F&& launch) {
  const int U = D / 8, per = kThreads / U;
  const int64_t blocks = ((int64_t)T + per - 1) / per;
  for (int64_t b = 0; b < blocks; b += kBlocksPerLaunch)
    launch((unsigned)std::min(blocks - b, kBlocksPerLaunch), U, per, b * per);
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

Rows rows_of(const void* codes, int64_t ch, int64_t cn, const void* scales, int64_t sh, int64_t sn, int bits) {
  const int64_t e = bits == 16 ? 2 : 1;
  return Rows{static_cast<char*>(const_cast<void*>(codes)), static_cast<char*>(const_cast<void*>(scales)), ch * e, cn * e, sh, sn};
}

}  // namespace

}  // namespace rspx

using namespace rspx;

extern "C" int rspx_kv_write_mx(const void* k, int64_t skt, int64_t skh, const void* v, int64_t svt, int64_t svh,
                                const int32_t* slots, int T, int cap, void* k_codes, int64_t skch, int64_t skcn,
                                void* k_scales, int64_t sksh, int64_t sksn, void* v_codes, int64_t svch, int64_t svcn,
                                void* v_scales, int64_t svsh, int64_t svsn, int HK, int D, int format, void* stream) {
  if (const int rc = sizes_ok(T, cap, HK, D, format)) return rc;
  if (format == RSPX_BF16) return RSPX_EUNSUPPORTED;   // rspx_kv_write
  if (T == 0) return RSPX_OK;
  const Tokens tk{static_cast<uint16_t*>(const_cast<void*>(k)), skt, skh}, tv{static_cast<uint16_t*>(const_cast<void*>(v)), svt, svh};
  const Rows ck = rows_of(k_codes, skch, skcn, k_scales, sksh, sksn, format),
             cv = rows_of(v_codes, svch, svcn, v_scales, svsh, svsn, format);
  if (!slots) return RSPX_EINVAL;
  for (const int rc : {tokens_ok(tk), tokens_ok(tv), rows_ok(ck, D, format), rows_ok(cv, D, format)})
    if (rc) return rc;
  return by_rows(T, D, [&](unsigned n, int U, int per, int64_t first) {
    const auto kernel = format == RSPX_MXFP8 ? kv_write_mx_kernel<8> : kv_write_mx_kernel<4>;
    hipLaunchKernelGGL(kernel, dim3(n, HK), dim3(kThreads), 0, static_cast<hipStream_t>(stream), tk, tv, slots, T, cap, ck, cv,
                       U, per, first);
  });
}

extern "C" int rspx_kv_read(const void* k_codes, int64_t skch, int64_t skcn, const void* k_scales, int64_t sksh, int64_t sksn,
                            const void* v_codes, int64_t svch, int64_t svcn, const void* v_scales, int64_t svsh, int64_t svsn,
                            const int32_t* slots, int T, int cap, void* k, int64_t skt, int64_t skh, void* v, int64_t svt,
                            int64_t svh, int HK, int D, int format, void* stream) {
  if (const int rc = sizes_ok(T, cap, HK, D, format)) return rc;
  if (T == 0) return RSPX_OK;
  const Tokens tk{static_cast<uint16_t*>(k), skt, skh}, tv{static_cast<uint16_t*>(v), svt, svh};
  const Rows ck = rows_of(k_codes, skch, skcn, k_scales, sksh, sksn, format),
             cv = rows_of(v_codes, svch, svcn, v_scales, svsh, svsn, format);
  if (!slots) return RSPX_EINVAL;
  for (const int rc : {tokens_ok(tk), tokens_ok(tv), rows_ok(ck, D, format), rows_ok(cv, D, format)})
    if (rc) return rc;
  return by_rows(T, D, [&](unsigned n, int U, int per, int64_t first) {
    const auto kernel = format == RSPX_BF16 ? kv_read_kernel<16> : format == RSPX_MXFP8 ? kv_read_kernel<8> : kv_read_kernel<4>;
    hipLaunchKernelGGL(kernel, dim3(n, HK), dim3(kThreads), 0, static_cast<hipStream_t>(stream), ck, cv, slots, T, cap, tk, tv,
                       U, per, first);
  });
}
