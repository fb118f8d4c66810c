// Log probabilities of given tokens, entropy and the best alternatives of every row of
// fp32 vocabulary scores, for gfx950.
//
//   p_j = exp(x_j - lse),  lse = m + log z,  z = sum_j exp(x_j - m),  m = max_j x_j
//   given = x_t - lse,  entropy = -sum_j p_j log p_j = log z - sum_j e_j (x_j - m) / z
//
// over the columns outside an excluded range.  One read of the scores: a wave takes 1024
// columns of one row at a time into registers and leaves (m, z, u = sum e (x - m)) of each
// such step; a second launch joins a row's steps in 64 bits, in an order that V alone sets.
// How many steps a workgroup takes depends on the number of rows, no result does.
//
// The best pairs are a set under a total order (value, lowest index first, NaN the
// largest), so their selection may take any order.  Each wave keeps a list of candidates in
// LDS and the bound that a pair must pass to enter it, the top-th best found so far: most
// steps add few or none.  Where a step would add many (the first one, rising scores, ties) they
// are bounded first by what the best pairs of `top` lanes pass, found to 16 bits of the value by
// a search over ballots, or, where ties let more through than the list has room for, exactly:
// at most 16 of each of `top` lanes then pass.  Lists are cut to their best by counting.
//
// What bounds it: the read of the scores, where there are many (1500 rows of 151936, top 5:
// 911 MB in 190 us, 4.8 TB/s; torch's sum over them reads 4.0); for one row two launches and
// the selection's dependent steps (kernels 6.0 us without alternatives, 9.6 with one, 13.4 with 20).
#include "common.h"
#include "respect_amd.h"

namespace rspx {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;                       // elements per lane
constexpr int kSub = 64 * kPer;                // columns of a wave's step: the unit of the sums
constexpr int kChunk = 4 * kSub;               // columns of a workgroup's step
constexpr int kMaxTop = 64;
constexpr int kMaxV = 1 << 30;                 // columns are counted in 32 bits
constexpr int kGroups = 64;                    // groups of four threads
constexpr float kL2E = 1.44269504088896340736f;

// Four scores of a row that starts anywhere: rows of an odd vocabulary are read as they are, as
// fast as aligned ones (1000 rows, top 5: of 50257 60.8 us, of 50256 60.2).
typedef float row4 __attribute__((ext_vector_type(4), aligned(4)));

// The order of the pairs as one unsigned number: larger is better.
__device__ __forceinline__ uint64_t pair_key(float v, int j) {
  uint32_t u = __float_as_uint(v + 0.0f);                  // -0 and +0 tie
  u = u & 0x80000000u ? ~u : u | 0x80000000u;
  if (v != v) u = 0xffffffffu;
  return (uint64_t)u << 32 | (0xffffffffu - (uint32_t)j);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  if (u == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); }

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  return (uint64_t)__shfl_xor((uint32_t)(v >> 32), m) << 32 | (uint32_t)__shfl_xor((uint32_t)v, m);
}

struct Select {
  uint64_t group[kGroups];
  uint64_t bound;
  int n;
  uint64_t cand[kMaxTop * kPer * 4];           // top groups of at most 4 threads' kPer elements
};

// The `top` best of the workgroup's keys (kPer per thread, 0 = none), handed best first to
// out(rank, key); ranks past the number of keys get key 0.  All threads call it.
template <class F>
__device__ __forceinline__ void select_top(const uint64_t (&key)[kPer], int top, Select& S, F&& out) {
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) best = key[i] > best ? key[i] : best;
  for (int m = 1; m <= 2; m <<= 1) {
    const uint64_t o = shfl_xor64(best, m);
    best = o > best ? o : best;
  }
  if ((threadIdx.x & 3) == 0) S.group[threadIdx.x >> 2] = best;
  if (threadIdx.x == 0) S.n = 0, S.bound = 0;
  __syncthreads();
  if (threadIdx.x < kGroups) {
    const uint64_t mine = S.group[threadIdx.x];
    int r = 0;
#pragma unroll 16
    for (int i = 0; i < kGroups; ++i) r += S.group[i] > mine;
    if (r == top - 1 && mine != 0) S.bound = mine;         // keys differ: one thread at most
  }
  __syncthreads();
  const uint64_t bound = S.bound > 1 ? S.bound : 1;        // fewer groups than `top`: every key
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (key[i] >= bound) S.cand[atomicAdd(&S.n, 1)] = key[i];
  __syncthreads();
  const int n = S.n;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = S.cand[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += S.cand[j] > mine;
    if (r < top) out(r, mine);
  }
  for (int i = n + threadIdx.x; i < top; i += kThreads) out(i, (uint64_t)0);
  __syncthreads();
}

struct LogArgs {
  const float* x;
  const int64_t* tokens;
  float *given, *entropy, *values;
  int64_t* ids;
  float* stat;                 // [rows][4 chunks][3]: m, z, u of each kSub columns
  uint64_t* best;              // [rows][parts][top]
  int64_t sx;
  int V, chunks, parts, off, end, top, row0;   // parts: workgroups of a row
};

// Entries a wave's list has room for: its best, the at most kPer of each of `top` lanes that a
// tightened bound lets through, and a copy of the best.
__host__ __device__ __forceinline__ int list_room(int top) { return (kPer + 2) * top; }

// The wave's list of n <= (kPer + 1) top pairs cut to its `top` best, best first; returns the
// last one, the bound of what may still enter (0: fewer than `top`).  The LDS operations of
// a wave keep their order.
__device__ __forceinline__ uint64_t prune(uint64_t* list, int& n, int top) {
  const int lane = __lane_id();
  uint64_t* best = list + (kPer + 1) * top;
  for (int i = lane; i < n; i += 64) {
    const uint64_t mine = list[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += list[j] > mine;
    if (r < top) best[r] = mine;
  }
  __builtin_amdgcn_wave_barrier();
  n = min(n, top);
  if (lane < n) list[lane] = best[lane];
  __builtin_amdgcn_wave_barrier();
  return n < top ? 0 : best[top - 1];
}

// How many of the wave's keys pass the bound.
__device__ __forceinline__ int passing(const uint64_t (&key)[kPer], uint64_t bound) {
  int count = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) count += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] > bound));
  return count;
}

// Adds the wave's step x (columns j0 + 256 (i / 4) + i % 4, j0 the lane's own) to its list.
__device__ __forceinline__ void enlist(const float (&x)[kPer], int j0, int V, int top, uint64_t* list, int& n,
                                       uint64_t& bound) {
  uint64_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = j0 + 256 * (i / 4) + i % 4;
    key[i] = j < V ? pair_key(x[i], j) : 0;
  }
  if (n + passing(key, bound) > 3 * top) {
    // Many: bounded by what the best pairs of `top` lanes pass, to 16 bits of the value.
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) best = key[i] > best ? key[i] : best;
    uint32_t p = 0;
    for (int b = 15; b >= 0; --b) {
      const uint32_t t = p | 1u << b;
      if (__builtin_popcountll(__builtin_amdgcn_ballot_w64((uint32_t)(best >> 48) >= t)) >= top) p = t;
    }
    if (p && ((uint64_t)p << 48) - 1 > bound) bound = ((uint64_t)p << 48) - 1;
    if (n + passing(key, bound) > (kPer + 1) * top) {      // still too many: by the top-th best pair of the lanes
      if (n > top) {
        const uint64_t last = prune(list, n, top);
        if (last > bound) bound = last;
      }
      int r = 0;
#pragma unroll 4
      for (int l = 0; l < 64; ++l) {
        const uint64_t o = (uint64_t)__builtin_amdgcn_readlane((int)(best >> 32), l) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)best, l);
        r += o > best;
      }
      const uint64_t at = __builtin_amdgcn_ballot_w64(r == top - 1 && best != 0);   // keys differ: one lane at most
      if (at) {
        const int l = __builtin_ctzll(at);
        const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(best >> 32), l) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)best, l);
        if (o - 1 > bound) bound = o - 1;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint64_t in = __builtin_amdgcn_ballot_w64(key[i] > bound);
    if (in) {
      if (key[i] > bound)
        list[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0))] = key[i];
      n += __builtin_popcountll(in);
    }
  }
  if (n > 2 * top) {
    const uint64_t last = prune(list, n, top);
    if (last > bound) bound = last;
  }
}

// Workgroup (part, row): the part's chunks in order, wave w the w-th quarter of each.
template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_part_kernel(LogArgs A) {
  extern __shared__ __align__(16) uint64_t lists[];        // [4][list_room(top)]
  __shared__ int counts[4];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)A.row0 + blockIdx.y;
  const float* xr = A.x + row * A.sx;
  const int c0 = (int)((int64_t)blockIdx.x * A.chunks / A.parts), c1 = (int)((int64_t)(blockIdx.x + 1) * A.chunks / A.parts);
  uint64_t* list = lists + w * list_room(A.top);
  int n = 0;
  uint64_t bound = 0;
  float least = kNegInf;                                   // the bound's value
  f32x4 next[kPer / 4];
  auto load = [&](int c) {
    const int j0 = c * kChunk + w * kSub + 4 * lane;
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) {
      const int j = j0 + 256 * i;
      f32x4 v = {kNegInf, kNegInf, kNegInf, kNegInf};
      if (j + 3 < A.V) v = *reinterpret_cast<const row4*>(xr + j);
      else
        for (int e = 0; e < 4; ++e)
          if (j + e < A.V) v[e] = xr[j + e];
      next[i] = v;
    }
  };
  load(c0);
  for (int c = c0; c < c1; ++c) {
    const int s0 = c * kChunk + w * kSub, j0 = s0 + 4 * lane;
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = next[i / 4][i % 4];
    if (c + 1 < c1) load(c + 1);
    if (s0 < A.end && s0 + kSub > A.off) {                 // excluded columns among them
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int j = j0 + 256 * (i / 4) + i % 4;
        if (j >= A.off && j < A.end) x[i] = kNegInf;
      }
    }
    float mine = x[0];
    bool nan = x[0] != x[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) {
      mine = fmaxf(mine, x[i]);
      nan |= x[i] != x[i];
    }
    nan = __builtin_amdgcn_ballot_w64(nan) != 0;
    float m = mine;
    for (int k = 32; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
    // e^d by 2^(d log2 e).  A -inf counts as e^-200 = 0, so that it adds no inf * 0; a step
    // of -inf only (m itself) adds nothing.
    float z = 0.f, u = 0.f;
    const float from = m == kNegInf ? 0.f : m;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float d = fmaxf(x[i] - from, -200.f);
      const float e = fexp2(d * kL2E);
      z = z + e;
      u = __builtin_fmaf(e, d, u);
    }
    for (int k = 32; k >= 1; k >>= 1) {
      z = z + __shfl_xor(z, k);
      u = u + __shfl_xor(u, k);
    }
    if (lane < 3) {
      const bool odd = nan || m == __builtin_huge_valf();  // NaN, or inf - inf
      const float v = lane == 0 ? m : lane == 1 ? z : u;
      A.stat[((row * A.chunks + c) * 4 + w) * 3 + lane] = odd && lane > 0 ? __builtin_nanf("") : v;
    }
    if constexpr (TOP) {
      if (__builtin_amdgcn_ballot_w64(mine >= least) != 0 || nan) {
        enlist(x, j0, A.V, A.top, list, n, bound);
        least = bound == 0 ? kNegInf : key_value(bound);
      }
    }
  }
  if constexpr (TOP) {
    if (n > A.top && A.top > 24) prune(list, n, A.top);    // ranking long lists costs more than this
    if (lane == 0) counts[w] = n;
    __syncthreads();
    // The best of the four waves' lists, ranked by counting.
    uint64_t* out = A.best + (row * A.parts + blockIdx.x) * A.top;
    const int room = list_room(A.top), all = counts[0] + counts[1] + counts[2] + counts[3];
    for (int i = threadIdx.x; i < all; i += kThreads) {
      int from = 0, at = i;
      for (int k = 0; k < 3; ++k)
        if (from == k && at >= counts[k]) at -= counts[k], ++from;
      const uint64_t key = lists[from * room + at];
      int r = 0;
      for (int k = 0; k < 4; ++k) {
        const int m = counts[k];
#pragma unroll 8
        for (int j = 0; j < m; ++j) r += lists[k * room + j] > key;
      }
      if (r < A.top) out[r] = key;
    }
    for (int i = all + threadIdx.x; i < A.top; i += kThreads) out[i] = 0;
  }
}

// One workgroup per row: the sums of its steps in 64 bits, each thread every 256th and the
// threads in a fixed tree, and the best of its parts' lists.
template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogArgs A) {
  __shared__ float sm[4];
  __shared__ double sz[4], su[4];
  __shared__ Select S;
  __shared__ uint64_t kept[kMaxTop];
  const int64_t row = (int64_t)A.row0 + blockIdx.x;
  const float* st = A.stat + row * A.chunks * 12;
  const int steps = 4 * A.chunks, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint64_t* b = A.best + row * A.parts * A.top;
  const int n = TOP ? A.parts * A.top : 0;
  const uint64_t own = n <= kThreads && (int)threadIdx.x < n ? b[threadIdx.x] : 0;
  const int64_t t = A.tokens[row];
  const bool there = t >= 0 && t < A.V;
  const float xt = there && !(t >= A.off && t < A.end) ? A.x[row * A.sx + t] : kNegInf;

  float m = kNegInf;
  for (int i = threadIdx.x; i < steps; i += kThreads) m = fmaxf(m, st[3 * i]);
  for (int k = 32; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
  if (lane == 0) sm[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  double z = 0, u = 0;
  for (int i = threadIdx.x; i < steps; i += kThreads) {
    const float mi = st[3 * i], zi = st[3 * i + 1], ui = st[3 * i + 2];
    if (zi != zi) z = zi;                                  // and stays
    if (mi == kNegInf) continue;                           // nothing in it
    const double d = (double)mi - (double)m, a = exp(d);
    z += a * zi;
    u += a * (ui + d * zi);
  }
  for (int k = 32; k >= 1; k >>= 1) {
    z += __shfl_xor(z, k);
    u += __shfl_xor(u, k);
  }
  if (lane == 0) {
    sz[w] = z;
    su[w] = u;
  }
  __syncthreads();
  z = (sz[0] + sz[1]) + (sz[2] + sz[3]);
  u = (su[0] + su[1]) + (su[2] + su[3]);
  // log p = (x - m) - log z: m + log z is never formed, scores of 1e38 would swallow log z.
  const double lz = log(z);
  auto logp = [&](float v) { return v == kNegInf && z == z ? kNegInf : (float)(((double)v - (double)m) - lz); };
  if (threadIdx.x == 0) {
    // A row with nothing left: every probability is 0, and so is the entropy.
    A.entropy[row] = m == kNegInf && z == 0 ? 0.f : (float)(lz - u / z);
    A.given[row] = there ? logp(xt) : __builtin_nanf("");
  }
  if constexpr (TOP) {
    if (n <= kThreads) {                                   // few: ranked by counting
      if ((int)threadIdx.x < n) S.cand[threadIdx.x] = own;
      __syncthreads();
      if (own != 0) {
        int r = 0;
#pragma unroll 8
        for (int i = 0; i < n; ++i) r += S.cand[i] > own;
        if (r < A.top) kept[r] = own;
      }
      __syncthreads();
    } else {                                               // in rounds of kChunk, the best so far carried along
      bool begun = false;
      for (int at = 0; at < n;) {
        uint64_t key[kPer];
        const int room = begun ? kChunk - kMaxTop : kChunk;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int p = threadIdx.x + kThreads * i;
          key[i] = p < room ? (at + p < n ? b[at + p] : 0) : (begun && p - room < A.top ? kept[p - room] : 0);
        }
        __syncthreads();
        select_top(key, A.top, S, [&](int r, uint64_t k) { kept[r] = k; });
        at += room;
        begun = true;
      }
    }
    for (int i = threadIdx.x; i < A.top; i += kThreads) {
      A.values[row * A.top + i] = logp(key_value(kept[i]));
      A.ids[row * A.top + i] = key_index(kept[i]);
    }
  }
}

// Workgroups per row: about 4096 in all, 2048 where the lists are long, at most one per chunk.
// A workgroup that takes more steps has its lists filled once for all of them (1000 rows, top
// 50: 303 us with 8192 workgroups, 242 with 4096, 210 with 2048; 1500 rows, top 5: 192, 187,
// 194), fewer of them fill the device less evenly (64 rows, top 20: 26.5, 26.5, 33.9).
int parts_of(int M, int chunks, int top) {
  const int total = top > 24 ? 2048 : 4096;
  const int want = (total + M - 1) / M;
  return want < chunks ? want : chunks;
}

constexpr int kRowsPerLaunch = 65535;

}  // namespace

}  // namespace rspx

using namespace rspx;

extern "C" int64_t rspx_token_logprobs_workspace_bytes(int M, int V, int top) {
  if (M < 0 || V <= 0 || V > kMaxV || top < 0 || top > kMaxTop) return -1;
  const int64_t chunks = ((int64_t)V + kChunk - 1) / kChunk;
  return (int64_t)M * (8 * (int64_t)top * (M ? parts_of(M, (int)chunks, top) : 0) + 48 * chunks) + 8;
}

extern "C" int rspx_token_logprobs(const float* logits, int64_t sl, int M, int V, int off, int size, const int64_t* tokens,
                                   int top, float* given, float* entropy, float* values, int64_t* ids, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (M < 0 || V <= 0 || sl < V || off < 0 || size < 0 || top < 0 || top > V) return RSPX_EINVAL;
  if (top > kMaxTop || V > kMaxV) return RSPX_EUNSUPPORTED;
  if (M == 0) return RSPX_OK;
  if (!logits || !tokens || !given || !entropy || (top && (!values || !ids))) return RSPX_EINVAL;
  if (reinterpret_cast<uintptr_t>(logits) & 3u) return RSPX_EALIGN;
  if (!workspace || workspace_bytes < rspx_token_logprobs_workspace_bytes(M, V, top)) return RSPX_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 7u) return RSPX_EALIGN;
  LogArgs A;
  A.x = logits;
  A.tokens = tokens;
  A.given = given, A.entropy = entropy, A.values = values, A.ids = ids;
  A.sx = sl;
  A.V = V, A.off = off, A.top = top;
  A.end = (int)((int64_t)off + size < V ? off + size : V);
  A.chunks = (int)(((int64_t)V + kChunk - 1) / kChunk);
  A.parts = parts_of(M, A.chunks, top);
  A.best = static_cast<uint64_t*>(workspace);
  A.stat = reinterpret_cast<float*>(A.best + (int64_t)M * A.parts * top);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned bytes = 4 * 8 * (unsigned)list_room(top);
  for (A.row0 = 0; A.row0 < M;) {
    const int n = M - A.row0 < kRowsPerLaunch ? M - A.row0 : kRowsPerLaunch;
    if (top) {
      hipLaunchKernelGGL(logprobs_part_kernel<true>, dim3(A.parts, n), dim3(kThreads), bytes, s, A);
      hipLaunchKernelGGL(logprobs_join_kernel<true>, dim3(n), dim3(kThreads), 0, s, A);
    } else {
      hipLaunchKernelGGL(logprobs_part_kernel<false>, dim3(A.parts, n), dim3(kThreads), 0, s, A);
      hipLaunchKernelGGL(logprobs_join_kernel<false>, dim3(n), dim3(kThreads), 0, s, A);
    }
    if (M - A.row0 <= kRowsPerLaunch) break;
    A.row0 += kRowsPerLaunch;
  }
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}
