// Attention of one new token per sequence over a paged KV cache, for gfx950.
//
//   o[b, h] = sum_j softmax_j(scale q[b, h] . k_j) v_j,   j < lens[b],
//
// k_j / v_j the rows of pool slot table[b][j / page] * page + j % page, query head h on
// kv head h / G.
//
// A sequence of n keys is cut into splits of split_keys(n) keys, a function of n alone, so
// a sequence's result does not depend on the rest of the batch nor on where its pages lie.
// The lengths are known on the device only: as many workgroups as are resident at once list
// the splits there are and take them in turn, (split, kv head) by (split, kv head), each
// requesting the first tile of its next one before it joins the waves of the present one.
// (A grid over every split that the table has room for, most of which end at once: 218 us
// instead of 60 for 64 sequences of up to 8000 keys.)  A second launch joins a sequence's
// splits, where the table has room for more than one.
//
// The four waves of a workgroup take the split's 32-key tiles in turn.  Scores are
// S^T = K Q^T by v_mfma_f32_16x16x32_bf16 with the G heads of the group in the 16 columns
// (the unused ones are zero); each lane then holds four keys of one head, the softmax runs
// there in fp32 with a lazily moved reference maximum, and the probabilities are used in
// place as the B operand of O^T += V^T P^T, as two bf16 terms: p cut to bf16 and the rest
// rounded to it (2^-15 of p is lost at most; the second product costs nothing next to the
// memory traffic).  Both terms are positive, so that an infinite v gives no inf - inf.  V
// goes from registers through a wave-private LDS stage to be read transposed.
//
// What bounds it: the K/V bytes, read once, where there are enough of them (one sequence of
// 131072 keys and five shorter ones, 32 / 8 heads of 128: 822 MB in 149 us, 5.5 TB/s; 64
// sequences of up to 8000: 260 MB in 64 us); below that the chain of dependent reads --
// lengths, table, K/V, the second launch's partial sums (13 us for one sequence of 4097, whose
// 17 MB take 3.3 of them).  Splits of 128 keys: 67 us instead of 64 for the batch, of 512: 17
// instead of 13 for the one; at most 64 splits, or two tiles per wave requested at once: no
// difference.
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
constexpr int kSeqs = 1024;          // sequences of a launch
constexpr int kCUs = 256;
constexpr float kTau = 8.0f;         // log2 headroom before the reference maximum moves
constexpr float kTiny = 1.17549435e-38f;   // the smallest normal number
constexpr float kNone = -1e30f;      // reference maximum before the first key

// Keys per split of a sequence of n keys: a multiple of kSplitKeys.
__host__ __device__ __forceinline__ int split_keys(int n) {
  const unsigned per = ((unsigned)n + kMaxSplits - 1) / kMaxSplits;
  return per <= kSplitKeys ? kSplitKeys : (int)((per + kSplitKeys - 1) / kSplitKeys * kSplitKeys);
}
__host__ __device__ __forceinline__ int split_count(int n) {
  const unsigned k = (unsigned)split_keys(n);
  return (int)(((unsigned)n + k - 1) / k);
}
// The most splits that any length up to n gives.
__host__ __forceinline__ int split_bound(int64_t n) { return n >= (int64_t)kSplitKeys * kMaxSplits ? kMaxSplits : split_count((int)n); }

struct PagedArgs {
  const uint16_t *q, *k, *v;
  const int *table, *lens;
  uint16_t* out;
  float* po;                   // [B][H][smax][D]: a split's sums
  f32x2* pml;                  // [B][H][smax]: its m and l
  int64_t sqb, sqh, skh, skn, svh, svn, stb, sob, soh;
  int B, HK, G, pages, shift, width, smax;
  float c;                     // scale * log2(e)
};

// first[b]: the splits of sequences before b (one for a sequence without any, whose rows
// are written too), length[b]: lens[b]; returns the number of splits.  All 256 threads call it.
__device__ __forceinline__ int list_items(const int* lens, int B, int64_t cap, int* first, int* length) {
  __shared__ int waves[4];
  constexpr int kPer = kSeqs / 256;
  int cnt[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i;
    cnt[i] = 0;
    if (b < B) {
      const int n = lens[b];
      length[b] = n;
      cnt[i] = n <= 0 || n > cap ? 1 : split_count(n);
    }
    sum += cnt[i];
  }
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int run = sum;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const int o = __shfl_up(run, k);
    if (lane >= k) run += o;
  }
  if (lane == 63) waves[w] = run;
  __syncthreads();
  int at = run - sum;
  for (int i = 0; i < w; ++i) at += waves[i];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    first[threadIdx.x * kPer + i] = at;
    at += cnt[i];
  }
  if (threadIdx.x == 255) first[kSeqs] = at;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(first[kSeqs]);
}

// The sequence that split number i belongs to.
__device__ __forceinline__ int find_seq(const int* first, int B, int i) {
  int lo = 0, hi = B;                                      // first[lo] <= i < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

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

// A barrier that does not wait for the loads in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xc07f);   // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ float max4(float x) { return fmaxf(fmaxf(x, shfl_xor(x, 16)), fmaxf(shfl_xor(x, 32), shfl_xor(x, 48))); }
__device__ __forceinline__ float sum4(float x) {
  x = x + shfl_xor(x, 16);
  return x + shfl_xor(x, 32);
}

template <int D>
struct PagedGeom {
  static constexpr int kPerCU = D >= 256 ? 1 : D >= 128 ? 2 : D >= 64 ? 3 : 4;   // resident workgroups
};

// One split of one sequence for one kv head.
struct Item {
  int g, b, n, split, splits;
  int t, tend;                 // this wave's first tile, and the end of the split's
};

template <int D>
__global__ __launch_bounds__(256, PagedGeom<D>::kPerCU) void paged_attn_kernel(PagedArgs A) {
  constexpr int NQ = D / 32, DT = D / 16, U = D / 8;
  constexpr int VL = kTile * U / 64;                       // 16-byte loads of a V tile per lane
  __shared__ __align__(16) char stage[kWaves][kTile * D * 2];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ int first[kSeqs + 1], length[kSeqs];

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c16 = lane & 15, r4 = lane >> 4;
  const int64_t cap = (int64_t)A.width << A.shift;
  const int items = list_items(A.lens, A.B, cap, first, length) * A.HK;
  if ((int)blockIdx.x >= items) return;

  auto decode = [&](int i) {
    Item x;
    x.g = i % A.HK;
    x.b = find_seq(first, A.B, i / A.HK);
    x.split = i / A.HK - __builtin_amdgcn_readfirstlane(first[x.b]);
    x.n = __builtin_amdgcn_readfirstlane(length[x.b]);
    x.splits = x.t = x.tend = 0;
    if (x.n > 0 && x.n <= cap) {
      const int per = split_keys(x.n);
      x.splits = split_count(x.n);
      x.t = x.split * (per / kTile) + w;
      x.tend = ((int)min((int64_t)x.n, (int64_t)(x.split + 1) * per) + kTile - 1) / kTile;
    }
    return x;
  };
  // The pool slot of key 32 t + lane % 32; keys past the end give the last one's.  -1: the
  // page is none, and nothing of it is read.
  auto slot_of = [&](const Item& x, int t) {
    const int key = min(t * kTile + (lane & 31), x.n - 1);
    const int p = A.table[x.b * A.stb + (key >> A.shift)];
    return (unsigned)p < (unsigned)A.pages ? (p << A.shift) + (key & ((1 << A.shift) - 1)) : -1;
  };
  u32x4 kf[2][NQ], vf[VL];
  auto load = [&](const Item& x, int slot) {
    slot = max(slot, 0);
    const uint16_t* kb = A.k + x.g * A.skh;
    const uint16_t* vb = A.v + x.g * A.svh;
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
  // B operand of the scores: lane (c16, r4) holds head c16, head_dim 32 i + 8 r4 .. + 7.
  bf16x8 qf[NQ];
  auto load_q = [&](const Item& x) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      u32x4 y = {0, 0, 0, 0};
      if (c16 < A.G)
        y = *reinterpret_cast<const u32x4*>(A.q + x.b * A.sqb + (int64_t)(x.g * A.G + c16) * A.sqh + 32 * i + 8 * r4);
      qf[i] = __builtin_bit_cast(bf16x8, y);
    }
  };

  lds_char* st = (lds_char*)stage[w];
  Item cur = decode(blockIdx.x);
  int slot = -1;                                           // of the tile in kf and vf
  if (cur.t < cur.tend) {
    slot = slot_of(cur, cur.t);
    load_q(cur);
    load(cur, slot);
  }
  for (int item = blockIdx.x;;) {
    const int after = item + gridDim.x;
    Item nxt = cur;
    nxt.t = nxt.tend = 0;
    if (after < items) nxt = decode(after);
    const int nslot = nxt.t < nxt.tend ? slot_of(nxt, nxt.t) : -1;
    uint16_t* orow = A.out + cur.b * A.sob + (int64_t)cur.g * A.G * A.soh;

    float mref = kNone, lsum = 0.f;
    f32x4 acc[DT];
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool bad = cur.t < cur.tend && slot < 0;
    int ahead = cur.t + kWaves < cur.tend ? slot_of(cur, cur.t + kWaves) : -1;
    for (int t = cur.t; t < cur.tend; t += kWaves) {
      f32x4 s[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf[j][i]), qf[i], s[j], 0, 0, 0);
      }
      const int left = cur.n - t * kTile;                  // keys of the tile that exist
      if (left < kTile) {   // the repeated last row: its p of 0 times inf would be NaN
#pragma unroll
        for (int j = 0; j < VL; ++j)
          if ((64 * j + lane) / U >= left) vf[j] = u32x4{0, 0, 0, 0};
      }
      // The stage belongs to this wave, whose LDS operations keep their order: the reads of
      // the tile before are done before these writes land.
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int u = 64 * j + lane, key = u / U;
        *(__attribute__((address_space(3))) u32x4*)(st + 16 * (key * U + ((u % U) ^ vswizzle<D>(key)))) = vf[j];
      }
      if (t + kWaves < cur.tend) {
        bad |= ahead < 0;
        load(cur, ahead);
        ahead = t + 2 * kWaves < cur.tend ? slot_of(cur, t + 2 * kWaves) : -1;
      }

      // Lane (c16, r4): head c16, keys 16 j + 4 r4 + e of the tile.
      float x[8], mx = kNegInf;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = s[i / 4][i % 4];
        if (left < kTile && 16 * (i / 4) + 4 * r4 + i % 4 >= left) x[i] = kNegInf;
        mx = fmaxf(mx, x[i]);
      }
      if (__builtin_amdgcn_ballot_w64(mx * A.c > mref + kTau) != 0) {
        const float top = max4(mx) * A.c;
        const float mn = top > mref + kTau ? top : mref;   // rows that stay get a factor of exactly 1
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
        hi[i] = __builtin_amdgcn_perm(__float_as_uint(p1), __float_as_uint(p0), 0x07060302u);
        lo[i] = pack_bf16x2(fmaxf(p0 - bf16_lo(hi[i]), kTiny), fmaxf(p1 - bf16_hi(hi[i]), kTiny));
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
        const bf16x8 va = __builtin_bit_cast(bf16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, ph, acc[j], 0, 0, 0);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pl, acc[j], 0, 0, 0);
      }
    }
    if (nxt.t < nxt.tend) {   // on its way while this item's waves are joined
      load_q(nxt);
      load(nxt, nslot);
    }
    if (cur.splits == 0) {    // no keys: zeros; a length that does not fit: NaN
      for (int i = threadIdx.x; i < A.G * D; i += 256) orow[(i / D) * A.soh + i % D] = cur.n == 0 ? 0 : 0x7fc0;
    } else {
      if (__builtin_amdgcn_ballot_w64(bad) != 0) lsum = __builtin_nanf("");
      lsum = sum4(lsum);
      // The four waves' results, joined in wave order.  A wave's stage holds its [16][D] sums
      // (the tile's V has been read by this wave).
      float* so = reinterpret_cast<float*>(&stage[0][0]);
#pragma unroll
      for (int j = 0; j < DT; ++j) *reinterpret_cast<f32x4*>(so + (w * 16 + c16) * D + (16 * j + 4 * r4)) = acc[j];
      if (r4 == 0) {
        sm[w][c16] = mref;
        sl[w][c16] = lsum;
      }
      lds_barrier();
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
        if (cur.splits == 1) {
          orow[h * A.soh + d] = f32_to_bf16_rne(o / l);
        } else {
          const int64_t p = (((int64_t)cur.b * A.HK + cur.g) * A.G + h) * A.smax + cur.split;
          A.po[p * D + d] = o;
          if (d == 0) A.pml[p] = f32x2{m, l};
        }
      }
      lds_barrier();   // the stages and the waves' m and l have been read
    }
    if (after >= items) break;
    item = after;
    cur = nxt;
    slot = nslot;
  }
}

// One workgroup per (query head, sequence).  Every wave takes the splits' weights, lane s
// that of split s; then lanes of four columns each sum every (256 / (D / 4))-th split, and
// those sums are added in order.
template <int D>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs A) {
  constexpr int L = D / 4, P = 256 / L;
  __shared__ float wt[kMaxSplits];
  __shared__ __align__(16) f32x4 sums[P][L];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63;
  const int64_t p = ((int64_t)b * A.HK * A.G + h) * A.smax;
  const f32x2 held = lane < A.smax ? A.pml[p + lane] : f32x2{kNone, 0.f};   // beside the length
  const int n = A.lens[b];
  if (n <= 0 || n > ((int64_t)A.width << A.shift)) return;
  const int splits = split_count(n);
  if (splits == 1) return;
  const f32x2 ml = lane < splits ? held : f32x2{kNone, 0.f};
  const int c = threadIdx.x % L, part = threadIdx.x / L;
  constexpr int N = (kMaxSplits + P - 1) / P;
  f32x4 x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = part + P * i;
    x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s < splits) x[i] = *reinterpret_cast<const f32x4*>(A.po + (p + s) * D + 4 * c);
  }
  float m = ml[0];
  for (int k = 32; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
  const float a = fexp2(ml[0] - m);
  float l = ml[1] * a;
  for (int k = 32; k >= 1; k >>= 1) l = l + __shfl_xor(l, k);
  if (threadIdx.x < kMaxSplits) wt[threadIdx.x] = a;
  __syncthreads();
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = part + P * i;
    const float f = s < splits ? wt[s] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[i][e], f, o[e]);
  }
  sums[part][c] = o;
  __syncthreads();
  if (threadIdx.x < D) {
    float t = 0.f;
    for (int i = 0; i < P; ++i) t = t + sums[i][threadIdx.x / 4][threadIdx.x % 4];
    A.out[b * A.sob + h * A.soh + threadIdx.x] = f32_to_bf16_rne(t / l);
  }
}

template <int D>
int launch(PagedArgs A, int B, hipStream_t s) {
  for (int b0 = 0; b0 < B; b0 += kSeqs) {
    A.B = B - b0 < kSeqs ? B - b0 : kSeqs;
    const int64_t items = (int64_t)A.B * A.smax * A.HK;
    hipLaunchKernelGGL(paged_attn_kernel<D>, dim3((unsigned)(items < kCUs * PagedGeom<D>::kPerCU ? items : kCUs * PagedGeom<D>::kPerCU)), dim3(256), 0, s, A);
    if (A.smax > 1) hipLaunchKernelGGL(paged_join_kernel<D>, dim3(A.HK * A.G, A.B), dim3(256), 0, s, A);
    A.q += A.B * A.sqb;
    A.out += A.B * A.sob;
    A.table += A.B * A.stb;
    A.lens += A.B;
    A.po += (int64_t)A.B * A.HK * A.G * A.smax * D;
    A.pml += (int64_t)A.B * A.HK * A.G * A.smax;
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
  if (!head_dim_ok(D) || H / HK > 16 || HK > 4096) return RSPX_EUNSUPPORTED;   // items of a launch are counted in 32 bits
  if (B == 0) return RSPX_OK;
  if (!q || !kc || !vc || !lens || !out || (width && !table)) return RSPX_EINVAL;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (reinterpret_cast<uintptr_t>(out) & 1u) return RSPX_EALIGN;
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
  A.po = static_cast<float*>(workspace);
  A.sqb = sqb, A.sqh = sqh, A.skh = skh, A.skn = skn, A.svh = svh, A.svn = svn, A.stb = stb, A.sob = sob, A.soh = soh;
  A.HK = HK, A.G = H / HK, A.pages = pages, A.width = width;
  A.shift = __builtin_ctz((unsigned)page);
  const int smax = split_bound((int64_t)width * page);
  A.smax = smax < 1 ? 1 : smax;
  A.pml = reinterpret_cast<f32x2*>(A.po + (int64_t)B * H * A.smax * D);
  A.c = sm_scale * 1.44269504088896340736f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (D) {
    case 32: return launch<32>(A, B, s);
    case 64: return launch<64>(A, B, s);
    case 128: return launch<128>(A, B, s);
    default: return launch<256>(A, B, s);
  }
}
