// Rows of a paged KV cache moved and written, for gfx950.
//
//   rspx_kv_move   rows from slot to slot in every layer's K and V pool: the begun page of
//                  a forked sequence, the accepted path of a verified trie
//   rspx_kv_move_mx  the same of pools of codes and of their scales (mx.h), in one launch
//   rspx_kv_write  new K and V rows of one layer to their slots
//
// Copies only; what bounds them is the bytes of the rows.  kv_move stores past the caches, so
// that the copies of one row do not push it out between them: 32 sequences forked 4 times
// (24 layers, 8 heads of 128, 69 MB read and 277 written) 79 us, 4.4 TB/s; 125 with ordinary
// stores, 82 with four units per thread, 130 with loads past the caches too.  32 paths of 13
// moved rows (82 MB): 13.7 us.
#include <algorithm>

#include "common.h"
#include "respect_amd.h"

namespace rspx {

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 8;            // 16-byte units a thread holds at once

// Workgroup (group, head, tensor): the group's moves in order, kThreads * kBatch units (of 16
// bytes; of a row of scales fewer) at a time, all of them read before any is written.  A slot
// outside [0, cap) is neither read nor written.  Strides in bytes.
template <class Unit>
__device__ __forceinline__ void move_group(const uint64_t* bases, int64_t sh, int64_t sn, int U, int cap,
                                           const int* groups, const int* moves, int n_moves, int g0) {
  char* base = reinterpret_cast<char*>(bases[blockIdx.z]) + blockIdx.y * sh;
  const int first = max(groups[g0 + blockIdx.x], 0), last = min(groups[g0 + blockIdx.x + 1], n_moves);
  if (first >= last) return;
  const int64_t total = (int64_t)(last - first) * U;
  for (int64_t u0 = 0; u0 < total; u0 += kThreads * kBatch) {
    Unit buf[kBatch];
    char* to[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      to[i] = nullptr;
      const int64_t u = u0 + i * kThreads + threadIdx.x;
      if (u < total) {
        const int m = (int)(u / U), c = (int)(u - (int64_t)m * U);
        const int src = moves[2 * (int64_t)(first + m)], dst = moves[2 * (int64_t)(first + m) + 1];
        if (src >= 0 && src < cap && dst >= 0 && dst < cap) {
          buf[i] = *reinterpret_cast<const Unit*>(base + src * sn + (int)sizeof(Unit) * c);
          to[i] = base + dst * sn + (int)sizeof(Unit) * c;
        }
      }
    }
    __syncthreads();   // the batch has been read
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (to[i]) __builtin_nontemporal_store(buf[i], reinterpret_cast<Unit*>(to[i]));
  }
}

// Pools of codes, and behind them as many pools of their scales.
struct MxPools {
  const uint64_t* bases;
  int64_t sch, scn, ssh, ssn;
  int tensors, U, V, unit, cap;        // units of a row of codes, of scales; bytes of the latter
};
__device__ __forceinline__ void move_mx(const MxPools& p, const int* groups, const int* moves, int n_moves, int g0) {
  if ((int)blockIdx.z < p.tensors) move_group<u32x4>(p.bases, p.sch, p.scn, p.U, p.cap, groups, moves, n_moves, g0);
  else if (p.unit == 8) move_group<u32x2>(p.bases, p.ssh, p.ssn, p.V, p.cap, groups, moves, n_moves, g0);
  else if (p.unit == 4) move_group<uint32_t>(p.bases, p.ssh, p.ssn, p.V, p.cap, groups, moves, n_moves, g0);
  else if (p.unit == 2) move_group<uint16_t>(p.bases, p.ssh, p.ssn, p.V, p.cap, groups, moves, n_moves, g0);
  else move_group<uint8_t>(p.bases, p.ssh, p.ssn, p.V, p.cap, groups, moves, n_moves, g0);
}

__global__ __launch_bounds__(kThreads) void kv_move_kernel(const uint64_t* bases, int64_t sh, int64_t sn, int U, int cap,
                                                           const int* groups, const int* moves, int n_moves, int g0) {
  move_group<u32x4>(bases, sh, sn, U, cap, groups, moves, n_moves, g0);
}
__global__ __launch_bounds__(kThreads) void kv_move_mx_kernel(MxPools p, const int* groups, const int* moves, int n_moves, int g0) {
  move_mx(p, groups, moves, n_moves, g0);
}

// The lists among the kernel's arguments: no copy to the device ahead of the launch (one prompt
// forked 4 times, with its tables and the forks freed: 16.0 us instead of 24.2; 32 paths of 13
// moved rows: 36.5 instead of 44).
struct Values {
  int x[RSPX_VALUES];
};
__global__ __launch_bounds__(kThreads) void kv_move_values_kernel(const uint64_t* bases, int64_t sh, int64_t sn, int U, int cap,
                                                                  int n_groups, int n_moves, Values lists) {
  move_group<u32x4>(bases, sh, sn, U, cap, lists.x, lists.x + n_groups + 1, n_moves, 0);
}
__global__ __launch_bounds__(kThreads) void kv_move_mx_values_kernel(MxPools p, int n_groups, int n_moves, Values lists) {
  move_mx(p, lists.x, lists.x + n_groups + 1, n_moves, 0);
}

// Tables and slots of a few sequences, likewise (the two calls above: 12.0 us and 32).
__global__ __launch_bounds__(kThreads) void values_kernel(int* out, int n, Values values) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < n) out[i] = values.x[i];
}

__global__ __launch_bounds__(kThreads) void kv_write_kernel(const uint16_t* k, int64_t skt, int64_t skh, const uint16_t* v,
                                                            int64_t svt, int64_t svh, const int* slots, int cap,
                                                            uint16_t* ck, int64_t sckh, int64_t sckn, uint16_t* cv,
                                                            int64_t scvh, int64_t scvn, int U, int HK, int64_t first,
                                                            int64_t total) {
  const int64_t i = first + (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= total) return;
  const int64_t r = i / U;
  const int c = (int)(i - r * U), h = (int)(r % HK);
  const int64_t t = r / HK;
  const int slot = slots[t];
  if (slot < 0 || slot >= cap) return;
  const u32x4 a = *reinterpret_cast<const u32x4*>(k + t * skt + h * skh + 8 * c);
  const u32x4 b = *reinterpret_cast<const u32x4*>(v + t * svt + h * svh + 8 * c);
  *reinterpret_cast<u32x4*>(ck + h * sckh + slot * sckn + 8 * c) = a;
  *reinterpret_cast<u32x4*>(cv + h * scvh + slot * scvn + 8 * c) = b;
}

constexpr int kGroupsPerLaunch = 1 << 20;
constexpr int64_t kBlocksPerLaunch = 1 << 23;   // a grid dimension holds 2^32 threads

}  // namespace

}  // namespace rspx

using namespace rspx;

static int check_move(const uint64_t* bases, int n_tensors, int HK, int D, int64_t sh, int64_t sn, int cap,
                      const int32_t* groups, int n_groups, const int32_t* moves, int n_moves) {
  if (n_tensors < 0 || HK < 1 || D < 1 || cap < 0 || n_groups < 0 || n_moves < 0 || sn < D || sh < 0) return RSPX_EINVAL;
  if (D % 8 || HK > 65535 || n_tensors > 65535) return RSPX_EUNSUPPORTED;
  if (sh % 8 || sn % 8) return RSPX_EALIGN;
  if (n_groups > 0 && n_moves > 0 && n_tensors > 0 && (!bases || !groups || !moves)) return RSPX_EINVAL;
  return RSPX_OK;
}

static Values listed(const int32_t* groups, int n_groups, const int32_t* moves, int n_moves) {
  Values lists;
  std::copy(groups, groups + n_groups + 1, lists.x);
  std::copy(moves, moves + 2 * n_moves, lists.x + n_groups + 1);
  std::fill(lists.x + n_groups + 1 + 2 * n_moves, lists.x + RSPX_VALUES, 0);
  return lists;
}

extern "C" int rspx_kv_move_values(const uint64_t* bases, int n_tensors, int HK, int D, int64_t sh, int64_t sn, int cap,
                                   const int32_t* groups, int n_groups, const int32_t* moves, int n_moves, void* stream) {
  if (const int rc = check_move(bases, n_tensors, HK, D, sh, sn, cap, groups, n_groups, moves, n_moves)) return rc;
  if ((int64_t)n_groups + 1 + 2 * (int64_t)n_moves > RSPX_VALUES) return RSPX_EUNSUPPORTED;
  if (n_groups == 0 || n_moves == 0 || n_tensors == 0) return RSPX_OK;
  const Values lists = listed(groups, n_groups, moves, n_moves);
  hipLaunchKernelGGL(kv_move_values_kernel, dim3(n_groups, HK, n_tensors), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), bases, 2 * sh, 2 * sn, D / 8, cap, n_groups, n_moves, lists);
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

extern "C" int rspx_values(const int32_t* values, int n, int32_t* out, void* stream) {
  if (n < 0) return RSPX_EINVAL;
  if (n > RSPX_VALUES) return RSPX_EUNSUPPORTED;
  if (n == 0) return RSPX_OK;
  if (!values || !out) return RSPX_EINVAL;
  if (reinterpret_cast<uintptr_t>(out) & 3u) return RSPX_EALIGN;
  Values v;
  std::fill(std::copy(values, values + n, v.x), v.x + RSPX_VALUES, 0);
  hipLaunchKernelGGL(values_kernel, dim3((n + kThreads - 1) / kThreads), dim3(kThreads), 0, static_cast<hipStream_t>(stream),
                     out, n, v);
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

extern "C" int rspx_kv_move(const uint64_t* bases, int n_tensors, int HK, int D, int64_t sh, int64_t sn, int cap,
                            const int32_t* groups, int n_groups, const int32_t* moves, int n_moves, void* stream) {
  if (const int rc = check_move(bases, n_tensors, HK, D, sh, sn, cap, groups, n_groups, moves, n_moves)) return rc;
  if (n_groups == 0 || n_moves == 0 || n_tensors == 0) return RSPX_OK;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for (int g0 = 0; g0 < n_groups; g0 += kGroupsPerLaunch) {
    const int n = n_groups - g0 < kGroupsPerLaunch ? n_groups - g0 : kGroupsPerLaunch;
    hipLaunchKernelGGL(kv_move_kernel, dim3(n, HK, n_tensors), dim3(kThreads), 0, s, bases, 2 * sh, 2 * sn, D / 8, cap, groups,
                       moves, n_moves, g0);
  }
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

// The checks of rspx_kv_move_mx*; fills p.
static int check_move_mx(const uint64_t* bases, int n_tensors, int HK, int D, int format, int64_t sch, int64_t scn, int64_t ssh,
                         int64_t ssn, int cap, const int32_t* groups, int n_groups, const int32_t* moves, int n_moves, MxPools& p) {
  if (format != RSPX_MXFP8 && format != RSPX_MXFP4) return RSPX_EUNSUPPORTED;
  if (n_tensors < 0 || HK < 1 || D < 1 || cap < 0 || n_groups < 0 || n_moves < 0 || sch < 0 || ssh < 0) return RSPX_EINVAL;
  if (D % 32 || HK > 65535 || n_tensors > 32767) return RSPX_EUNSUPPORTED;
  const int row = D * format / 8, scales = D / 32;
  if (scn < row || ssn < scales) return RSPX_EINVAL;
  if (sch % 16 || scn % 16) return RSPX_EALIGN;
  if (n_groups > 0 && n_moves > 0 && n_tensors > 0 && (!bases || !groups || !moves)) return RSPX_EINVAL;
  int unit = 8;
  while (scales % unit || ssh % unit || ssn % unit) unit /= 2;
  p = MxPools{bases, sch, scn, ssh, ssn, n_tensors, row / 16, scales / unit, unit, cap};
  return RSPX_OK;
}

extern "C" int rspx_kv_move_mx(const uint64_t* bases, int n_tensors, int HK, int D, int format, int64_t sch, int64_t scn,
                               int64_t ssh, int64_t ssn, int cap, const int32_t* groups, int n_groups, const int32_t* moves,
                               int n_moves, void* stream) {
  MxPools p;
  if (const int rc = check_move_mx(bases, n_tensors, HK, D, format, sch, scn, ssh, ssn, cap, groups, n_groups, moves, n_moves, p))
    return rc;
  if (n_groups == 0 || n_moves == 0 || n_tensors == 0) return RSPX_OK;
  for (int g0 = 0; g0 < n_groups; g0 += kGroupsPerLaunch)
    hipLaunchKernelGGL(kv_move_mx_kernel, dim3(std::min(n_groups - g0, kGroupsPerLaunch), HK, 2 * n_tensors), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), p, groups, moves, n_moves, g0);
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

extern "C" int rspx_kv_move_mx_values(const uint64_t* bases, int n_tensors, int HK, int D, int format, int64_t sch, int64_t scn,
                                      int64_t ssh, int64_t ssn, int cap, const int32_t* groups, int n_groups,
                                      const int32_t* moves, int n_moves, void* stream) {
  MxPools p;
  if (const int rc = check_move_mx(bases, n_tensors, HK, D, format, sch, scn, ssh, ssn, cap, groups, n_groups, moves, n_moves, p))
    return rc;
  if ((int64_t)n_groups + 1 + 2 * (int64_t)n_moves > RSPX_VALUES) return RSPX_EUNSUPPORTED;
  if (n_groups == 0 || n_moves == 0 || n_tensors == 0) return RSPX_OK;
  hipLaunchKernelGGL(kv_move_mx_values_kernel, dim3(n_groups, HK, 2 * n_tensors), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), p, n_groups, n_moves, listed(groups, n_groups, moves, n_moves));
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

extern "C" int rspx_kv_write(const void* k, int64_t skt, int64_t skh, const void* v, int64_t svt, int64_t svh,
                             const int32_t* slots, int T, int cap, void* cache_k, int64_t sckh, int64_t sckn,
                             void* cache_v, int64_t scvh, int64_t scvn, int HK, int D, void* stream) {
  if (T < 0 || cap < 0 || HK < 1 || D < 1 || sckn < D || scvn < D) return RSPX_EINVAL;
  if (D % 8) return RSPX_EUNSUPPORTED;
  if (T == 0) return RSPX_OK;
  if (!k || !v || !slots || !cache_k || !cache_v) return RSPX_EINVAL;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (!al(k) || !al(v) || !al(cache_k) || !al(cache_v)) return RSPX_EALIGN;
  for (int64_t x : {skt, skh, svt, svh, sckh, sckn, scvh, scvn})
    if (x % 8) return RSPX_EALIGN;
  const int U = D / 8;
  const int64_t total = (int64_t)T * HK * U, blocks = (total + kThreads - 1) / kThreads;
  for (int64_t b0 = 0; b0 < blocks; b0 += kBlocksPerLaunch)
    hipLaunchKernelGGL(kv_write_kernel, dim3((unsigned)std::min(blocks - b0, kBlocksPerLaunch)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), static_cast<const uint16_t*>(k), skt, skh,
                       static_cast<const uint16_t*>(v), svt, svh, slots, cap, static_cast<uint16_t*>(cache_k), sckh, sckn,
                       static_cast<uint16_t*>(cache_v), scvh, scvn, U, HK, b0 * kThreads, total);
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}
