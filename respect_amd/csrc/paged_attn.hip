// Attention of one new token per sequence over a paged KV cache, for gfx950.
//
//   o[b, h] = sum_j softmax_j(scale q[b, h] . k_j) v_j,   j < lens[b],
//
// k_j / v_j the rows of pool slot table[b][j / page] * page + j % page, query head h on
// kv head h / G.  One launch over (split, kv head, sequence), and a second one that joins
// the splits where a sequence may have more than one.
//
// A sequence of n keys is cut into splits of split_keys(n) keys, a function of n alone, so
// a sequence's result does not depend on the rest of the batch nor on where its pages lie.
// The four waves of a workgroup take the split's 32-key tiles in turn.  Scores are
// S^T = K Q^T by v_mfma_f32_16x16x32_bf16 with the G heads of the group in the 16 columns
// (the unused ones are zero); each lane then holds four keys of one head, the softmax runs
// there in fp32 with a lazily moved reference maximum, and the probabilities are used in
// place as the B operand of O^T += V^T P^T, as bf16 hi + lo (relative error 2^-17: the
// product costs nothing next to the memory traffic, so they are not cut to bf16).  V goes
// from registers through a wave-private LDS stage to be read transposed.
//
// What bounds it: the K/V bytes; nothing is read twice.
#include <type_traits>

#include "common.h"
#include "respect_amd.h"

namespace rspx {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kTile = 32;            // keys of a wave's step
constexpr int kWaves = 4;
constexpr int kSplitKeys = 256;      // the shortest split
constexpr int kMaxSplits = 32;       // a longer cache gets longer splits
constexpr float kTau = 8.0f;         // log2 headroom before the reference maximum moves
constexpr float kNone = -1e30f;      // reference maximum before the first key

// Keys per split of a sequence of n keys: a multiple of kSplitKeys.
__host__ __device__ __forceinline__ int split_keys(int n) {
  const int per = (int)(((int64_t)n + kMaxSplits - 1) / kMaxSplits);
  return per <= kSplitKeys ? kSplitKeys : (per + kSplitKeys - 1) / kSplitKeys * kSplitKeys;
}
__host__ __device__ __forceinline__ int split_count(int n) {
  const int k = split_keys(n);
  return (int)(((int64_t)n + k - 1) / k);
}
// The most splits that any length up to n gives.
__host__ __forceinline__ int split_bound(int64_t n) { return n >= (int64_t)kSplitKeys * kMaxSplits ? kMaxSplits : split_count((int)n); }

struct PagedArgs {
  const uint16_t *q, *k, *v;
  const int *table, *lens;
  uint16_t* out;
  float* part;                 // [B][H][smax][D + 2]: O, then m, l
  int64_t sqb, sqh, skh, skn, svh, svn, stb, sob, soh;
  int HK, G, pages, shift, width, smax;
  float c;                     // scale * log2(e)
};

__device__ __forceinline__ s16x4 tr_read(const lds_char* __restrict__ p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
}

// 16-byte unit swizzle of a staged V row: four consecutive keys' pairs of units lie in
// different banks for the transposing reads.
template <int D>
__device__ __forceinline__ int vswizzle(int key) {
  constexpr int U = D / 8;
  if constexpr (U >= 16) return 2 * (key % 8);
  else return 2 * ((key / (16 / U)) % (U / 2));
}

__device__ __forceinline__ float max4(float x) { return fmaxf(fmaxf(x, shfl_xor(x, 16)), fmaxf(shfl_xor(x, 32), shfl_xor(x, 48))); }
__device__ __forceinline__ float sum4(float x) {
  x = x + shfl_xor(x, 16);
  return x + shfl_xor(x, 32);
}

template <int D>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedArgs A) {
  constexpr int NQ = D / 32, DT = D / 16, U = D / 8;
  constexpr int VL = kTile * U / 64;                       // 16-byte loads of a V tile per lane
  __shared__ __align__(16) char stage[kWaves][kTile * D * 2];
  __shared__ float sm[kWaves][16], sl[kWaves][16];

  const int split = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
  const int n = A.lens[b];
  const int page = 1 << A.shift;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, r4 = lane >> 4;
  const int64_t cap = (int64_t)A.width << A.shift;
  uint16_t* orow = A.out + b * A.sob + (int64_t)g * A.G * A.soh;
  if (n <= 0 || n > cap) {                                 // no keys: zeros; a length that does not fit: NaN
    if (split == 0)
      for (int i = threadIdx.x; i < A.G * D; i += 256) orow[(i / D) * A.soh + i % D] = n == 0 ? 0 : 0x7fc0;
    return;
  }
  const int per = split_keys(n), splits = split_count(n);
  if (split >= splits) return;
  const int tend = (min(n, (split + 1) * per) + kTile - 1) / kTile;
  const int tfirst = split * (per / kTile) + w;

  // B operand of the scores: lane (c16, r4) holds head c16, head_dim 32 i + 8 r4 .. + 7.
  bf16x8 qf[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    u32x4 x = {0, 0, 0, 0};
    if (c16 < A.G)
      x = *reinterpret_cast<const u32x4*>(A.q + b * A.sqb + (int64_t)(g * A.G + c16) * A.sqh + 32 * i + 8 * r4);
    qf[i] = __builtin_bit_cast(bf16x8, x);
  }

  const int* row = A.table + b * A.stb;
  const uint16_t* kb = A.k + g * A.skh;
  const uint16_t* vb = A.v + g * A.svh;
  bool bad = false;
  // The pool slot of key 32 t + lane % 32; keys past the end give the last one's.
  auto slot_of = [&](int tile) {
    const int key = min(tile * kTile + (lane & 31), n - 1);
    int p = row[key >> A.shift];
    if ((unsigned)p >= (unsigned)A.pages) {                // a page that is none: nothing of it is read
      bad = true;
      p = 0;
    }
    return (p << A.shift) + (key & (page - 1));
  };
  u32x4 kf[2][NQ], vf[VL];
  auto load = [&](int slot) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint16_t* p = kb + shfl_idx_i(slot, 16 * j + c16) * A.skn + 8 * r4;
#pragma unroll
      for (int i = 0; i < NQ; ++i) kf[j][i] = *reinterpret_cast<const u32x4*>(p + 32 * i);
    }
#pragma unroll
    for (int j = 0; j < VL; ++j) {
      const int u = 64 * j + lane;
      vf[j] = *reinterpret_cast<const u32x4*>(vb + shfl_idx_i(slot, u / U) * A.svn + 8 * (u % U));
    }
  };

  lds_char* st = (lds_char*)stage[w];
  float mref, lsum;
  f32x4 acc[DT];
  auto pass = [&](auto odd) {
    mref = kNone, lsum = 0.f;
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int t = tfirst;
    int slot = t < tend ? slot_of(t) : 0;
    if (t < tend) load(slot);
    int next = t + kWaves < tend ? slot_of(t + kWaves) : 0;
    for (; t < tend; t += kWaves) {
      f32x4 s[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf[j][i]), qf[i], s[j], 0, 0, 0);
      }
      // The stage belongs to this wave, whose LDS operations keep their order: the reads of
      // the tile before are done before these writes land.
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int u = 64 * j + lane, key = u / U;
        *(__attribute__((address_space(3))) u32x4*)(st + 16 * (key * U + ((u % U) ^ vswizzle<D>(key)))) = vf[j];
      }
      if (t + kWaves < tend) {
        load(next);
        next = t + 2 * kWaves < tend ? slot_of(t + 2 * kWaves) : 0;
      }

      // Lane (c16, r4): head c16, keys 16 j + 4 r4 + e of the tile.
      const int left = n - t * kTile;                        // keys of the tile that exist
      float x[8], mx = kNegInf;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = s[i / 4][i % 4];
        if (left < kTile && 16 * (i / 4) + 4 * r4 + i % 4 >= left) x[i] = kNegInf;
        mx = fmaxf(mx, x[i]);
      }
      if (__builtin_amdgcn_ballot_w64(mx * A.c > mref + kTau) != 0) {
        const float top = max4(mx) * A.c;
        const float mn = top > mref + kTau ? top : mref;     // rows that stay get a factor of exactly 1
        const float alpha = fexp2(mref - mn);
        lsum = lsum * alpha;
        mref = mn;
#pragma unroll
        for (int j = 0; j < DT; ++j) acc[j] = acc[j] * alpha;
      }
      u32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p0 = fexp2(__builtin_fmaf(x[2 * i], A.c, -mref)), p1 = fexp2(__builtin_fmaf(x[2 * i + 1], A.c, -mref));
        lsum = lsum + p0;
        lsum = lsum + p1;
        hi[i] = pack_bf16x2(p0, p1);
        lo[i] = pack_bf16x2(p0 - bf16_lo(hi[i]), p1 - bf16_hi(hi[i]));
      }
      const bf16x8 ph = __builtin_bit_cast(bf16x8, hi), pl = __builtin_bit_cast(bf16x8, lo);
      // A operand of head_dim tile j: V[key(k)][16 j + c16], k-slots 8 r4 + i <-> keys
      // 4 r4 + i (i < 4) and 12 + 4 r4 + i, the order in which the lane holds p.
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        s16x4 h[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int key = 16 * z + 4 * r4 + (c16 >> 2), u = 2 * j + ((c16 & 3) >> 1);
          h[z] = tr_read(st + 16 * (key * U + (u ^ vswizzle<D>(key))) + 8 * (c16 & 1));
        }
        if (left < kTile) {   // the repeated last row: 0 * inf would be NaN
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (16 * (i / 4) + 4 * r4 + i % 4 >= left) h[i / 4][i % 4] = 0;
        }
        const bf16x8 va = __builtin_bit_cast(bf16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, ph, acc[j], 0, 0, 0);
        if constexpr (odd) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if ((h[i / 4][i % 4] & 0x7f80) == 0x7f80) h[i / 4][i % 4] = 0;
        }
        const bf16x8 vl = __builtin_bit_cast(bf16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vl, pl, acc[j], 0, 0, 0);
      }
    }
  };
  pass(std::false_type());
  // lo * v is 0 * inf or -inf for an infinite v: a wave whose sums are not finite takes its
  // tiles again, without such values in the lo product (the other columns keep their bits).
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 4 * DT; ++i) finite &= __builtin_fabsf(acc[i / 4][i % 4]) < __builtin_huge_valf();
  if (__builtin_amdgcn_ballot_w64(!finite) != 0) pass(std::true_type());
  if (__builtin_amdgcn_ballot_w64(bad) != 0) lsum = __builtin_nanf("");
  lsum = sum4(lsum);

  // The four waves' results, joined in wave order.  A wave's stage holds its [16][D] sums
  // (the tile's V has been read by this wave).
  float* so = reinterpret_cast<float*>(&stage[0][0]);
#pragma unroll
  for (int j = 0; j < DT; ++j)
    *reinterpret_cast<f32x4*>(so + (w * 16 + c16) * D + (16 * j + 4 * r4)) = acc[j];
  if (r4 == 0) {
    sm[w][c16] = mref;
    sl[w][c16] = lsum;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < A.G * D; i += 256) {
    const int h = i / D, d = i % D;
    float m = sm[0][h];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) m = fmaxf(m, sm[k][h]);
    float o = 0.f, l = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float a = fexp2(sm[k][h] - m);
      l = __builtin_fmaf(sl[k][h], a, l);
      o = __builtin_fmaf(so[(k * 16 + h) * D + d], a, o);
    }
    if (splits == 1) {
      orow[h * A.soh + d] = f32_to_bf16_rne(o / l);
    } else {
      float* p = A.part + (((int64_t)b * A.HK + g) * A.G + h) * A.smax * (D + 2) + (int64_t)split * (D + 2);
      p[d] = o;
      if (d == 0) {
        p[D] = m;
        p[D + 1] = l;
      }
    }
  }
}

// One workgroup per (query head, sequence): the splits in order, one column per thread.
template <int D>
__global__ __launch_bounds__(D) void paged_join_kernel(PagedArgs A) {
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const int n = A.lens[b];
  if (n <= 0 || n > ((int64_t)A.width << A.shift)) return;
  const int splits = split_count(n);
  if (splits == 1) return;
  const float* p = A.part + ((int64_t)b * A.HK * A.G + h) * A.smax * (D + 2);
  float m = p[D];
  for (int s = 1; s < splits; ++s) m = fmaxf(m, p[s * (D + 2) + D]);
  float o = 0.f, l = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float a = fexp2(p[s * (D + 2) + D] - m);
    l = __builtin_fmaf(p[s * (D + 2) + D + 1], a, l);
    o = __builtin_fmaf(p[s * (D + 2) + d], a, o);
  }
  A.out[b * A.sob + h * A.soh + d] = f32_to_bf16_rne(o / l);
}

constexpr int kGridZ = 65535;   // sequences of a launch

template <int D>
int launch(PagedArgs A, int B, hipStream_t s) {
  for (int b0 = 0; b0 < B; b0 += kGridZ) {
    const int nb = B - b0 < kGridZ ? B - b0 : kGridZ;
    hipLaunchKernelGGL(paged_attn_kernel<D>, dim3(A.smax, A.HK, nb), dim3(256), 0, s, A);
    if (A.smax > 1) hipLaunchKernelGGL(paged_join_kernel<D>, dim3(A.HK * A.G, nb), dim3(D), 0, s, A);
    A.q += nb * A.sqb;
    A.out += nb * A.sob;
    A.table += nb * A.stb;
    A.lens += nb;
    A.part += (int64_t)nb * A.HK * A.G * A.smax * (D + 2);
  }
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

bool head_dim_ok(int D) { return D == 32 || D == 64 || D == 128 || D == 256; }

}  // namespace

}  // namespace rspx

using namespace rspx;

extern "C" int64_t rspx_paged_attn_workspace_bytes(int B, int H, int D, int page, int width) {
  if (B < 0 || H < 1 || page < 1 || width < 0 || !head_dim_ok(D)) return -1;
  const int smax = split_bound((int64_t)width * page);
  return smax <= 1 ? 0 : (int64_t)B * H * smax * (D + 2) * 4;
}

extern "C" int rspx_paged_attn(const void* q, int64_t sqb, int64_t sqh, const void* kc, int64_t skh, int64_t skn,
                               const void* vc, int64_t svh, int64_t svn, const int32_t* table, int64_t stb,
                               const int32_t* lens, void* out, int64_t sob, int64_t soh, int B, int H, int HK, int D,
                               int pages, int page, int width, float sm_scale, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  if (B < 0 || H < 1 || HK < 1 || H % HK || pages < 1 || page < 1 || (page & (page - 1)) || width < 0) return RSPX_EINVAL;
  if (!(sm_scale > 0.f) || sm_scale > 3e38f) return RSPX_EINVAL;
  if ((int64_t)pages * page > INT32_MAX || (int64_t)width * page > INT32_MAX - 4096) return RSPX_EINVAL;
  if (!head_dim_ok(D) || H / HK > 16 || HK > 65535) return RSPX_EUNSUPPORTED;
  if (B == 0) return RSPX_OK;
  if (!q || !kc || !vc || !lens || !out || (width && !table)) return RSPX_EINVAL;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (!al(q) || !al(kc) || !al(vc) || sqb % 8 || sqh % 8 || skh % 8 || skn % 8 || svh % 8 || svn % 8) return RSPX_EALIGN;
  const int64_t need = rspx_paged_attn_workspace_bytes(B, H, D, page, width);
  if (need > 0 && (!workspace || workspace_bytes < need)) return RSPX_EWORKSPACE;
  if (need > 0 && !al(workspace)) return RSPX_EALIGN;
  PagedArgs A;
  A.q = static_cast<const uint16_t*>(q);
  A.k = static_cast<const uint16_t*>(kc);
  A.v = static_cast<const uint16_t*>(vc);
  A.table = table;
  A.lens = lens;
  A.out = static_cast<uint16_t*>(out);
  A.part = static_cast<float*>(workspace);
  A.sqb = sqb, A.sqh = sqh, A.skh = skh, A.skn = skn, A.svh = svh, A.svn = svn, A.stb = stb, A.sob = sob, A.soh = soh;
  A.HK = HK, A.G = H / HK, A.pages = pages, A.width = width;
  A.shift = __builtin_ctz((unsigned)page);
  const int smax = split_bound((int64_t)width * page);
  A.smax = smax < 1 ? 1 : smax;
  A.c = sm_scale * 1.44269504088896340736f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (D) {
    case 32: return launch<32>(A, B, s);
    case 64: return launch<64>(A, B, s);
    case 128: return launch<128>(A, B, s);
    default: return launch<256>(A, B, s);
  }
}
