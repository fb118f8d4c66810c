// Log probabilities of given tokens, entropy and the best alternatives of every row of
// fp32 vocabulary scores, for gfx950.
//
//   p_j = exp(x_j - lse),  lse = m + log z,  z = sum_j exp(x_j - m),  m = max_j x_j
//   given = x_t - lse,  entropy = -sum_j p_j log p_j = log z - sum_j e_j (x_j - m) / z
//
// over the columns outside an excluded range.  One read of the scores: a workgroup takes a
// chunk of kChunk columns of one row into registers, leaves the chunk's (m, z, u = sum e (x - m))
// and its best `top` (value, index) pairs, and a second launch joins a row's chunks in
// order, in 64 bits.  A row's result depends on its own scores and on V alone.
//
// The best pairs are a set under a total order (value, lowest index first, NaN the
// largest), so their selection may take any order: the top-th best of 64 groups' maxima is a
// lower bound of the top-th best element, what passes it (at most 64 per group that does, in
// practice a few more than `top`) is gathered and ranked by counting.
//
// What bounds it: the read of the scores.
#include "common.h"
#include "respect_amd.h"

namespace rspx {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;                       // elements per thread
constexpr int kChunk = kThreads * kPer;        // columns of a workgroup
constexpr int kMaxTop = 64;
constexpr int kGroups = 64;                    // groups of four threads

// exp(x) for x <= 0 (or NaN): x log2(e) in two pieces, so that the product's rounding does
// not grow with |x|.
__device__ __forceinline__ float exp_neg(float x) {
  constexpr float kL = 1.44269504088896340736f, kLlo = 1.92596299e-8f, kLn2 = 0.69314718055994530942f;
  const float h = x * kL;
  const float l = __builtin_fmaf(x, kLlo, __builtin_fmaf(x, kL, -h));
  const float e = fexp2(h);
  return x < -100.f ? e : __builtin_fmaf(e, l * kLn2, e);   // -inf: no inf - inf in l
}

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
  float* stat;                 // [rows][chunks][3]: m, z, u
  uint64_t* best;              // [rows][chunks][top]
  int64_t sx;
  int V, chunks, off, end, top, row0;
};

__device__ __forceinline__ bool excluded(const LogArgs& A, int j) { return j >= A.off && j < A.end; }

__device__ __forceinline__ float block_max(float v, float* s) {
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_chunk_kernel(LogArgs A) {
  __shared__ float sm[4], sz[4], su[4];
  __shared__ Select S;
  const int c = blockIdx.x;
  const int64_t row = (int64_t)A.row0 + blockIdx.y;
  const float* xr = A.x + row * A.sx;
  float x[kPer];
#pragma unroll
  for (int i = 0; i < kPer / 4; ++i) {
    const int j = c * kChunk + 4 * (threadIdx.x + kThreads * i);
    f32x4 v = {kNegInf, kNegInf, kNegInf, kNegInf};
    if (j + 3 < A.V) v = *reinterpret_cast<const f32x4*>(xr + j);
    else
      for (int e = 0; e < 4; ++e)
        if (j + e < A.V) v[e] = xr[j + e];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = excluded(A, j + e) ? kNegInf : v[e];
  }
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) m = fmaxf(m, x[i]);
  m = block_max(m, sm);
  float z = 0.f, u = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float d = m == kNegInf ? x[i] : x[i] - m;        // a chunk of -inf adds nothing
    const float e = exp_neg(d);
    z = z + e;
    u = u + (d == kNegInf ? 0.f : e * d);
  }
  for (int k = 32; k >= 1; k >>= 1) {
    z = z + __shfl_xor(z, k);
    u = u + __shfl_xor(u, k);
  }
  if ((threadIdx.x & 63) == 0) {
    sz[threadIdx.x >> 6] = z;
    su[threadIdx.x >> 6] = u;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    float* st = A.stat + (row * A.chunks + c) * 3;
    st[0] = m;
    st[1] = (sz[0] + sz[1]) + (sz[2] + sz[3]);
    st[2] = (su[0] + su[1]) + (su[2] + su[3]);
  }
  if constexpr (TOP) {
    uint64_t key[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = c * kChunk + 4 * (threadIdx.x + kThreads * (i / 4)) + i % 4;
      key[i] = j < A.V ? pair_key(x[i], j) : 0;
    }
    uint64_t* b = A.best + (row * A.chunks + c) * A.top;
    select_top(key, A.top, S, [&](int r, uint64_t k) { b[r] = k; });
  }
}

// One workgroup per row.
template <bool TOP>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogArgs A) {
  __shared__ double slz;
  __shared__ float smax;
  __shared__ Select S;
  __shared__ uint64_t kept[kMaxTop];
  const int64_t row = (int64_t)A.row0 + blockIdx.x;
  if (threadIdx.x == 0) {
    const float* st = A.stat + row * A.chunks * 3;
    float m = kNegInf;
    for (int c = 0; c < A.chunks; ++c) m = fmaxf(m, st[3 * c]);
    double z = 0, u = 0;
    for (int c = 0; c < A.chunks; ++c) {
      const double d = (double)st[3 * c] - (double)m;
      if (st[3 * c] == kNegInf && !(st[3 * c + 1] != st[3 * c + 1])) continue;   // nothing in it, no NaN either
      const double a = exp(d);
      z += a * st[3 * c + 1];
      u += a * (st[3 * c + 2] + d * st[3 * c + 1]);
    }
    const double lz = log(z);
    // A row with nothing left: every probability is 0, and so is the entropy.
    A.entropy[row] = m == kNegInf && z == 0 ? 0.f : (float)(lz - u / z);
    const int64_t t = A.tokens[row];
    float given = __builtin_nanf("");                      // no such token
    if (t >= 0 && t < A.V) {
      const float x = excluded(A, (int)t) ? kNegInf : A.x[row * A.sx + t];
      given = x == kNegInf && z == z ? kNegInf : (float)(((double)x - (double)m) - lz);
    }
    A.given[row] = given;
    slz = lz;   // lse = m + lz is never formed: scores of 1e38 would swallow lz
    smax = m;
  }
  if constexpr (TOP) {
    // The chunks' best in rounds of kChunk keys, the best so far carried along.
    const uint64_t* b = A.best + row * A.chunks * A.top;
    const int n = A.chunks * A.top;
    int at = 0;
    bool first = true;
    while (first || at < n) {
      uint64_t key[kPer];
      const int room = first ? kChunk : kChunk - kMaxTop;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int p = threadIdx.x + kThreads * i;
        key[i] = p < room ? (at + p < n ? b[at + p] : 0) : (!first && p - room < A.top ? kept[p - room] : 0);
      }
      __syncthreads();
      select_top(key, A.top, S, [&](int r, uint64_t k) { kept[r] = k; });
      at += room;
      first = false;
    }
    for (int i = threadIdx.x; i < A.top; i += kThreads) {
      const float v = key_value(kept[i]);
      A.values[row * A.top + i] = v == kNegInf && slz == slz ? kNegInf : (float)(((double)v - (double)smax) - slz);
      A.ids[row * A.top + i] = key_index(kept[i]);
    }
  }
}

constexpr int kRowsPerLaunch = 65535;

}  // namespace

}  // namespace rspx

using namespace rspx;

extern "C" int64_t rspx_token_logprobs_workspace_bytes(int M, int V, int top) {
  if (M < 0 || V <= 0 || top < 0 || top > kMaxTop) return -1;
  const int64_t chunks = ((int64_t)V + kChunk - 1) / kChunk;
  return (int64_t)M * chunks * (8 * (int64_t)top + 12) + 8;
}

extern "C" int rspx_token_logprobs(const float* logits, int64_t sl, int M, int V, int off, int size, const int64_t* tokens,
                                   int top, float* given, float* entropy, float* values, int64_t* ids, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (M < 0 || V <= 0 || sl < V || off < 0 || size < 0 || top < 0 || top > V) return RSPX_EINVAL;
  if (top > kMaxTop) return RSPX_EUNSUPPORTED;
  if (M == 0) return RSPX_OK;
  if (!logits || !tokens || !given || !entropy || (top && (!values || !ids))) return RSPX_EINVAL;
  if ((reinterpret_cast<uintptr_t>(logits) & 15u) || sl % 4) return RSPX_EALIGN;
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
  A.best = static_cast<uint64_t*>(workspace);
  A.stat = reinterpret_cast<float*>(A.best + (int64_t)M * A.chunks * top);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for (A.row0 = 0; A.row0 < M;) {
    const int n = M - A.row0 < kRowsPerLaunch ? M - A.row0 : kRowsPerLaunch;
    if (top) {
      hipLaunchKernelGGL(logprobs_chunk_kernel<true>, dim3(A.chunks, n), dim3(kThreads), 0, s, A);
      hipLaunchKernelGGL(logprobs_join_kernel<true>, dim3(n), dim3(kThreads), 0, s, A);
    } else {
      hipLaunchKernelGGL(logprobs_chunk_kernel<false>, dim3(A.chunks, n), dim3(kThreads), 0, s, A);
      hipLaunchKernelGGL(logprobs_join_kernel<false>, dim3(n), dim3(kThreads), 0, s, A);
    }
    if (M - A.row0 <= kRowsPerLaunch) break;
    A.row0 += kRowsPerLaunch;
  }
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}
