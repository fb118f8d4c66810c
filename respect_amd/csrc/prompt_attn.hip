// Causal attention over whole prompts, packed one after the other, for gfx950.
//
//   o[t, h] = sum_j softmax_j(scale q[t, h] . k_j) v_j
//
// over the keys j that row t of its sequence sees.  The work is a list of tiles of at most
// 32 RW rows of one sequence; a workgroup takes one tile for 4 / RW query heads of one kv
// head, each wave 32 rows of one head.  Keys and values of 64 positions at a time go from
// memory straight into LDS (two slots of each) and serve all four waves.
//
// A wave computes S^T = K Q^T by v_mfma_f32_32x32x16_bf16, so a lane holds 32 scores of one
// row: the softmax (fp32, a running maximum that moves only when a score passes it by
// 2^kTau) needs no lane exchange but the rare move's.  The probabilities, rounded to bf16
// as the trie attention rounds them (half a step each), are summed in fp32 as rounded, so that
// numerator and denominator weigh alike, and used in place as the B operand of O^T += V^T P^T
// with V read transposed from LDS.  In steps that every row sees whole, the next step's score
// products and this step's exponentials, then the products with V and the next maximum, stand
// alternating in the code: four simple instructions or two exponentials cost nothing beside a
// product of the same wave.
//
// Every row is computed from its own column of the MFMA tiles in 64-key steps from the
// sequence's first key on: its bits depend on its sequence alone, not on the pack, on the
// tile it falls in or on later rows.
//
// What bounds it: in long prompts the power budget (16384 tokens, 32 / 8 heads of 128: 1.86 to
// 1.97 ms by the card, 1.12 to 1.18 PFLOP/s, where a large library product reaches 1.41; the
// clock is down to 1.7 GHz, the MFMAs are busy 65 % of it, VALU half; the LDS reads, 128 KB per
// step and workgroup, take half as long as the MFMAs, without bank conflicts); in packed prompts
// besides it the starts and ends of the workgroups; in short ones and few heads what one wave
// per SIMD issues in a step (0.87 us at D = 128, of which the MFMAs are 0.48; memory has no part
// in it: keys that all lie in one row take as long).  The order of the whole steps, held by
// scheduling barriers, took 3 % off the long cases (the compiler's own: 1.93 ms beside 1.87, 24
// packed prompts 278 us beside 270) and nothing off the short; addresses worked out once and
// probabilities summed in pairs 2 to 3 % off these (219 instructions a step instead of 268).
// Measured and not kept: eight waves per tile that take the steps in turn and are joined
// (three quarters of the time with few workgroups, but 337 us instead of 289 for 24 packed
// prompts, and the choice may not depend on the pack), three and four steps in LDS (no
// gain), the compiler's own interleaving groups (5 to 30 % slower), wave priorities (2 %),
// whole steps not unrolled by two, which copies the scores (270 -> 278 us), and the barrier in
// the middle of a step, operands of the next one requested before its end (0 to 2 %).
#include <algorithm>

#include "common.h"
#include "respect_amd.h"

namespace rspx {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kKeys = 64;            // keys of a step
constexpr int kRows = 32;            // rows of a wave
constexpr float kTau = 8.0f;         // log2 headroom before the reference maximum moves
constexpr float kNone = -1e30f;      // reference maximum before the first key

constexpr int kGroups = 1 << 23;     // workgroups of a launch: a grid dimension holds 2^32 threads
constexpr int kEdges = 8;            // more than the steps that some row of a tile sees in part
// Waves per SIMD, that is workgroups per CU, that the registers and the LDS allow.
constexpr int waves_per_simd(int D) { return D >= 256 ? 1 : D >= 128 ? 2 : D >= 64 ? 3 : 4; }

struct PromptArgs {
  const uint16_t *q, *k, *v;
  const int* tiles;            // [n][4]: first row, rows, first key, keys the first row sees
  uint16_t* out;
  int64_t sqt, sqh, skt, skh, svt, svh, sot, soh;
  int G, Tq, Tk, units;        // units = H / heads per workgroup
  float c;                     // scale * log2(e)
};

// Non-template wrappers: the host pass rejects these builtins inside templates.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, uint32_t nbytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)nbytes, 0x00020000);
}
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t r, int voff, lds_char* dst) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 16, voff, 0, 0, 0);
}
__device__ __forceinline__ s16x4 tr_read(const lds_char* __restrict__ p) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
}

typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
// c + both bf16 of x, rounded to nearest (measured: 63 of 64 sums as one rounding, none by more
// than 0.52 of a step).
__device__ __forceinline__ float dot2(uint32_t x, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b16x2, x), __builtin_bit_cast(b16x2, 0x3f803f80u), c, false);
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

// HW heads and RW = 4 / HW row blocks of 32 rows per workgroup.
template <int D, int HW>
__global__ __launch_bounds__(256, waves_per_simd(D)) void prompt_attn_kernel(PromptArgs A) {
  constexpr int U = D / 8, NS = D / 16, DT = D / 32;
  constexpr int kBytes = kKeys * D * 2;                    // K or V of one step
  constexpr int kLoads = kBytes / 1024 / 4;                // 1 KB loads per wave, K and V each
  // One object: beside a second one the compiler waits for the loads to LDS in flight, the
  // next step's too, ahead of a step's first read.
  __shared__ __align__(16) char lds[4 * kBytes + 4 * kEdges];
  int* flags = reinterpret_cast<int*>(lds + 4 * kBytes);

  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int unit = blockIdx.x % A.units, tile = blockIdx.x / A.units;
  const int head = unit * HW + w % HW;
  const int kvh = (unit * HW) / A.G;
  const int* T = A.tiles + 4 * (int64_t)tile;
  // A tile that points outside the tensors is cut to them.
  const int q0 = min(max(T[0], 0), A.Tq), k0 = min(max(T[2], 0), A.Tk);
  const int rows = min(min(max(T[1], 0), kRows * (4 / HW)), A.Tq - q0);
  const int seen0 = T[3];                                  // row i sees keys [k0, k0 + seen0 + i)
  const int keys = (int)min(max((int64_t)seen0 + rows - 1, (int64_t)0), (int64_t)(A.Tk - k0));
  const int steps = (keys + kKeys - 1) / kKeys;
  const int whole = min(max(seen0, 0), keys) / kKeys;      // steps that every row sees whole
  if (threadIdx.x < kEdges) flags[threadIdx.x] = 0;

  const int rb = kRows * (w / HW);                         // this wave's rows in the tile
  const int row = rb + col;
  const int seen = (int)min((int64_t)seen0 + row, (int64_t)keys);   // keys of this lane's row
  const bool live = row < rows;

  // B operand of the scores: lane (col, half) holds row col, head_dim 16 i + 8 half .. + 7.
  bf16x8 qf[NS];
  const uint16_t* qrow = A.q + (int64_t)(q0 + (live ? row : 0)) * A.sqt + (int64_t)head * A.sqh + 8 * half;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    u32x4 x = {0, 0, 0, 0};
    if (live) x = *reinterpret_cast<const u32x4*>(qrow + 16 * i);
    qf[i] = __builtin_bit_cast(bf16x8, x);
  }

  // Byte offsets of this lane's units of a step's K and V: load j of wave w fills units
  // 64 (4 j + w) + lane of the stage.  Rows past the last key read as zeros.
  const uint16_t* kp = A.k + (int64_t)k0 * A.skt + (int64_t)kvh * A.skh;
  const uint16_t* vp = A.v + (int64_t)k0 * A.svt + (int64_t)kvh * A.svh;
  int ko[kLoads], vo[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int u = 64 * (4 * j + w) + lane, key = u / U;
    ko[j] = (int)(2 * key * A.skt) + 16 * ((u % U) ^ kswizzle<D>(key));
    vo[j] = (int)(2 * key * A.svt) + 16 * ((u % U) ^ vswizzle<D>(key));
  }
  auto issue_k = [&](int t) {
    if (t >= steps) return;
    const int left = min(keys - t * kKeys, kKeys);
    const auto r = rsrc(kp + (int64_t)t * kKeys * A.skt, (uint32_t)(2 * (left - 1) * A.skt + 2 * D));
    lds_char* dst = (lds_char*)lds + kBytes * (t & 1);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) to_lds(r, ko[j], dst + 1024 * (4 * j + w));
  };
  auto issue_v = [&](int t) {
    if (t >= steps) return;
    const int left = min(keys - t * kKeys, kKeys);
    const auto r = rsrc(vp + (int64_t)t * kKeys * A.svt, (uint32_t)(2 * (left - 1) * A.svt + 2 * D));
    lds_char* dst = (lds_char*)lds + kBytes * (2 + (t & 1));
#pragma unroll
    for (int j = 0; j < kLoads; ++j) to_lds(r, vo[j], dst + 1024 * (4 * j + w));
  };
  // Byte offsets in a step's K and V of this lane's first operands: those of the others differ
  // by constants, added for keys and xored, as the swizzles are, for head_dim.  Made once: the
  // compiler would work them out anew in every step.
  int k_at = 16 * (col * U + (half ^ kswizzle<D>(col)));
  int v_at;
  {
    const int l16 = lane & 15, key = 4 * half + (l16 >> 2), u = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
    v_at = 16 * (key * U + (u ^ vswizzle<D>(key))) + 8 * (l16 & 1);
  }
  asm("" : "+v"(k_at), "+v"(v_at));
  // A operand of the scores: keys 32 kb + col, head_dim 16 i + 8 half .. + 7.
  auto kread = [&](const lds_char* sk, int i, int kb) __attribute__((always_inline)) {
    return __builtin_bit_cast(bf16x8, read16(sk + (k_at ^ (32 * i)) + 16 * 32 * U * kb));
  };
  // S^T of a step: two blocks of 32 keys.  Lane (col, half): row col, keys 32 kb + 8 (e / 4) + 4 half + e % 4.
  auto scores = [&](int t, f32x16 (&o)[2]) __attribute__((always_inline)) {
    const lds_char* sk = (const lds_char*)lds + kBytes * (t & 1);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[kb][e] = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        o[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kread(sk, i, kb), qf[i], o[kb], 0, 0, 0);
  };
  f32x16 s[2], next[2];
  if (steps > 0) {
    issue_k(0);
    issue_v(0);
    __builtin_amdgcn_s_waitcnt(0x0F70 | kLoads);           // vmcnt(kLoads): this wave's part of K
    lds_barrier();
    issue_k(1);
    scores(0, s);
  }

  float mref = kNone, lsum = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int j = 0; j < DT; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;

  // A operand of head_dim tile j, 16-key step i: V[key][32 j + lane % 32], k-slots
  // 8 half + e <-> keys 16 i + 8 (e / 4) + 4 half + e % 4, the order in which the lane holds p.
  auto vread = [&](const lds_char* sv, int i, int j) __attribute__((always_inline)) {
    s16x4 h[2];
#pragma unroll
    for (int z = 0; z < 2; ++z) h[z] = tr_read(sv + (v_at ^ (64 * j)) + 16 * U * (16 * i + 8 * z));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // The running maximum moved, and what hangs on it, where a row's largest score passes it.
  auto move = [&](float mx) __attribute__((always_inline)) {
    if (__builtin_amdgcn_ballot_w64(mx * A.c > mref + kTau) != 0) {
      const float top = fmaxf(mx, shfl_xor(mx, 32)) * A.c;
      const float mn = top > mref + kTau ? top : mref;     // rows that stay get a factor of exactly 1
      const float alpha = fexp2(mref - mn);
      lsum = lsum * alpha;
      mref = mn;
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[j][e] = acc[j][e] * alpha;
    }
  };
  // Two probabilities of the row, of scores r and r + 1, as bf16.
  auto pair = [&](const f32x16 (&s)[2], int r) __attribute__((always_inline)) {
    const float a = fexp2(__builtin_fmaf(s[r / 16][r % 16], A.c, -mref));
    const float b = fexp2(__builtin_fmaf(s[r / 16][r % 16 + 1], A.c, -mref));
    const uint32_t x = pack_bf16x2(a, b);
    lsum = dot2(x, lsum);
    return x;
  };

  const int first_edge = min(whole, steps - 1);            // the last step has no scores to run ahead
  // One step that every row sees whole, its scores in s and the maximum moved; the next
  // step's scores come to `next`.  In program order, which the barriers keep: a matrix
  // product, the operands of the third after it, and as much of the softmax as fits beside it.
  auto whole_step = [&](int t, const f32x16 (&s)[2], f32x16 (&next)[2]) __attribute__((always_inline)) {
    constexpr int NA = 2 * NS, NB = 4 * DT, Z = 3;
    __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0): this wave's part of V and the next K
    lds_barrier();                                         // everyone's; and the step before is read
    issue_k(t + 2);
    issue_v(t + 1);
    const lds_char* sk = (const lds_char*)lds + kBytes * ((t + 1) & 1);
    const lds_char* sv = (const lds_char*)lds + kBytes * (2 + (t & 1));
    bf16x8 x[Z + 1];
    u32x4 p[4];
#pragma unroll
    for (int n = 0; n < Z; ++n) x[n] = kread(sk, n / 2, n % 2);
    f32x16 zero;
#pragma unroll
    for (int e = 0; e < 16; ++e) zero[e] = 0.f;
    // The next scores beside the first half of the exponentials.
#pragma unroll
    for (int n = 0; n < NA; ++n) {
      if (n + Z < NA) x[(n + Z) % (Z + 1)] = kread(sk, (n + Z) / 2, (n + Z) % 2);
      else x[(n + Z) % (Z + 1)] = vread(sv, (n + Z - NA) / DT, (n + Z - NA) % DT);
      next[n % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[n % (Z + 1)], qf[n / 2], n < 2 ? zero : next[n % 2], 0, 0, 0);
#pragma unroll
      for (int i = 8 * n / NA; i < 8 * (n + 1) / NA; ++i) p[i / 4][i % 4] = pair(s, 2 * i);
      __builtin_amdgcn_sched_barrier(0);
    }
    // The product with V beside the other half, then beside the next scores' maximum.
    float mx = kNegInf;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if (n + Z < NB) x[(NA + n + Z) % (Z + 1)] = vread(sv, (n + Z) / DT, (n + Z) % DT);
      acc[n % DT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[(NA + n) % (Z + 1)], __builtin_bit_cast(bf16x8, p[n / DT]),
                                                            acc[n % DT], 0, 0, 0);
      if (n < NB / 2) {
#pragma unroll
        for (int i = 8 + 16 * n / NB; i < 8 + 16 * (n + 1) / NB; ++i) p[i / 4][i % 4] = pair(s, 2 * i);
      } else {
#pragma unroll
        for (int i = 64 * (n - NB / 2) / NB; i < 64 * (n - NB / 2 + 1) / NB; ++i) mx = fmaxf(mx, next[i / 16][i % 16]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (t + 1 < first_edge) move(mx);
  };
  // One step of 64 keys that some row may not see all of, or the last one; its scores are in s.
  auto edge_step = [&](int t) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0): this wave's part of V and the next K
    lds_barrier();                                         // everyone's; and the step before is read
    issue_k(t + 2);
    issue_v(t + 1);
    lds_char* sv = (lds_char*)lds + kBytes * (2 + (t & 1));
    // A key that a row does not see has p = 0, but 0 * inf and 0 * NaN are NaN: such a value
    // among the step's may not reach the rows before it.  Each wave looks a quarter of V over.
    uint32_t found = 0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const u32x4 x = read16(sv + 1024 * (4 * j + w) + 16 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) found |= (x[e] & 0x7f807f80u) + 0x00800080u;   // an exponent of ones carries
    }
    if (__builtin_amdgcn_ballot_w64((found & 0x80008000u) != 0) != 0 && lane == 0) flags[t - first_edge] = 1;
    lds_barrier();

    const int mine = seen - t * kKeys;                     // keys of the step that this lane's row sees
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (32 * kb + 8 * (e / 4) + 4 * half + e % 4 >= mine) s[kb][e] = kNegInf;
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) mx = fmaxf(mx, s[i / 16][i % 16]);
    move(mx);
    u32x4 p[4];
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i / 4][i % 4] = pair(s, 2 * i);
    if (__builtin_amdgcn_readfirstlane(flags[t - first_edge]) != 0) {
      // The values that are not finite go to the rows that see them one by one, and the
      // product runs without them: every other sum keeps its bits.  Where p is 0 they are NaN,
      // as the product makes them in a step seen whole (its registers cost the whole steps 0.3 to
      // 0.5 %: 5 packed prompts of 7577 tokens 182.6 us instead of 181.7).
      uint32_t none[2] = {0, 0};                           // scores with p = 0, of this lane and the row's other one
#pragma unroll
      for (int r = 0; r < 32; ++r)
        if ((p[r / 8][r / 2 % 4] >> (16 * (r % 2)) & 0xffffu) == 0) none[0] |= 1u << r;
      none[1] = (uint32_t)__shfl_xor((int)none[0], 32);
#pragma unroll 1
      for (int key = 0; key < kKeys; ++key) {
        const int r = 16 * (key / 32) + 4 * (key % 32 / 8) + key % 4;   // key's place among its lane's scores
        const bool zero = (none[key / 4 % 2 != half] >> r & 1) != 0;
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int d = 32 * j + 8 * (e / 4) + 4 * half + e % 4;
            const uint16_t x = *(const __attribute__((address_space(3))) uint16_t*)(
                sv + 16 * (key * U + ((d / 8) ^ vswizzle<D>(key))) + 2 * (d % 8));
            if ((x & 0x7f80) == 0x7f80 && key < mine) acc[j][e] = acc[j][e] + (zero ? __builtin_nanf("") : bf16_to_f32(x));
          }
      }
      lds_barrier();
#pragma unroll 1
      for (int j = 0; j < kLoads; ++j) {
        auto* at = (__attribute__((address_space(3))) u32x4*)(sv + 1024 * (4 * j + w) + 16 * lane);
        u32x4 x = *at;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u;
          if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0xffffu;
        }
        *at = x;
      }
      lds_barrier();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < DT; ++j)
        acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vread(sv, i, j), __builtin_bit_cast(bf16x8, p[i]), acc[j], 0, 0, 0);
    if (t + 1 < steps) scores(t + 1, s);
  };

  int t = 0;
  if (first_edge > 0) {
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) mx = fmaxf(mx, s[i / 16][i % 16]);
    move(mx);
  }
  for (; t + 1 < first_edge; t += 2) {                     // the scores change places: no copies
    whole_step(t, s, next);
    whole_step(t + 1, next, s);
  }
  if (t < first_edge) {
    whole_step(t, s, next);
    s[0] = next[0], s[1] = next[1];
    ++t;
  }
  for (; t < steps; ++t) edge_step(t);

  // Lane (col, half): row col, head_dim 32 j + 8 (e / 4) + 4 half + e % 4.
  if (!live) return;
  lsum = lsum + shfl_xor(lsum, 32);
  const float inv = 1.0f / lsum;
  uint16_t* o = A.out + (int64_t)(q0 + row) * A.sot + (int64_t)head * A.soh + 4 * half;
#pragma unroll
  for (int j = 0; j < DT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u32x2 x;
#pragma unroll
      for (int z = 0; z < 2; ++z) x[z] = pack_bf16x2(acc[j][4 * e + 2 * z] * inv, acc[j][4 * e + 2 * z + 1] * inv);
      if (seen <= 0) x = u32x2{0, 0};                      // a row that sees no key
      *reinterpret_cast<u32x2*>(o + 32 * j + 8 * e) = x;
    }
}

int heads_per_group(int G) { return G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1; }

template <int D>
int launch(PromptArgs A, int HW, int n, hipStream_t s) {
  const int per = kGroups / A.units;
  for (; n > 0; n -= per, A.tiles += 4 * (int64_t)per) {
    const dim3 grid((unsigned)(A.units * std::min(n, per)));
    if (HW == 4) hipLaunchKernelGGL((prompt_attn_kernel<D, 4>), grid, dim3(256), 0, s, A);
    else if (HW == 2) hipLaunchKernelGGL((prompt_attn_kernel<D, 2>), grid, dim3(256), 0, s, A);
    else hipLaunchKernelGGL((prompt_attn_kernel<D, 1>), grid, dim3(256), 0, s, A);
  }
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

}  // namespace

}  // namespace rspx

using namespace rspx;

extern "C" int rspx_prompt_attn_tile_rows(int H, int HK) {
  if (H < 1 || HK < 1 || H % HK) return -1;
  return kRows * (4 / heads_per_group(H / HK));
}

extern "C" int64_t rspx_prompt_attn_tiles(const int64_t* rows, const int64_t* keys, int n, int tile_rows, int32_t* tiles) {
  if (n < 0 || tile_rows < 1 || (n > 0 && (!rows || !keys))) return RSPX_EINVAL;
  int64_t tq = 0, tk = 0, count = 0;
  for (int i = 0; i < n; ++i) {
    if (rows[i] < 0 || keys[i] < 0 || rows[i] > INT32_MAX || keys[i] > INT32_MAX) return RSPX_EINVAL;
    tq += rows[i], tk += keys[i], count += (rows[i] + tile_rows - 1) / tile_rows;
    if (tq > INT32_MAX || tk > INT32_MAX) return RSPX_EINVAL;
  }
  if (!tiles) return count;
  struct Tile {
    int32_t x[4];
  };
  Tile* out = reinterpret_cast<Tile*>(tiles);
  tq = tk = count = 0;
  for (int i = 0; i < n; ++i) {
    for (int64_t r = 0; r < rows[i]; r += tile_rows) {
      const int64_t m = rows[i] - r < tile_rows ? rows[i] - r : tile_rows;
      out[count++] = Tile{{(int32_t)(tq + r), (int32_t)m, (int32_t)tk, (int32_t)(keys[i] - rows[i] + r + 1)}};
    }
    tq += rows[i], tk += keys[i];
  }
  // The longest first, so that the device is busy to the end (ties: in the order of the rows).
  std::sort(out, out + count, [](const Tile& a, const Tile& b) {
    const int64_t x = (int64_t)a.x[1] + a.x[3], y = (int64_t)b.x[1] + b.x[3];
    return x != y ? x > y : a.x[0] < b.x[0];
  });
  return count;
}

extern "C" int rspx_prompt_attn(const void* q, int64_t sqt, int64_t sqh, const void* k, int64_t skt, int64_t skh,
                                const void* v, int64_t svt, int64_t svh, const int32_t* tiles, int n_tiles, void* out,
                                int64_t sot, int64_t soh, int H, int HK, int Tq, int Tk, int D, float sm_scale,
                                void* stream) {
  if (H < 1 || HK < 1 || H % HK || Tq < 0 || Tk < 0 || n_tiles < 0) return RSPX_EINVAL;
  if (!(sm_scale > 0.f) || sm_scale > 3e38f) return RSPX_EINVAL;
  if (D != 32 && D != 64 && D != 128 && D != 256) return RSPX_EUNSUPPORTED;
  // Byte offsets inside a 64-key step are 32-bit.
  constexpr int64_t kMaxStride = 1 << 24;
  if (sqt < 0 || sqh < 0 || skt < 0 || skh < 0 || svt < 0 || svh < 0 || sot < 0 || soh < 0 || skt >= kMaxStride ||
      svt >= kMaxStride)
    return RSPX_EINVAL;
  if (n_tiles == 0 || Tq == 0) return RSPX_OK;
  if (!q || !tiles || !out || (Tk > 0 && (!k || !v))) return RSPX_EINVAL;
  auto al = [](const void* p, unsigned a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; };
  if (!al(q, 16) || !al(k, 16) || !al(v, 16) || !al(out, 8) || sqt % 8 || sqh % 8 || skt % 8 || skh % 8 || svt % 8 ||
      svh % 8 || sot % 4 || soh % 4)
    return RSPX_EALIGN;
  PromptArgs A;
  A.q = static_cast<const uint16_t*>(q);
  A.k = static_cast<const uint16_t*>(k);
  A.v = static_cast<const uint16_t*>(v);
  A.tiles = tiles;
  A.out = static_cast<uint16_t*>(out);
  A.sqt = sqt, A.sqh = sqh, A.skt = skt, A.skh = skh, A.svt = svt, A.svh = svh, A.sot = sot, A.soh = soh;
  A.G = H / HK, A.Tq = Tq, A.Tk = Tk;
  const int HW = heads_per_group(A.G);
  A.units = H / HW;
  if (A.units > kGroups) return RSPX_EUNSUPPORTED;
  A.c = sm_scale * 1.44269504088896340736f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (D) {
    case 32: return launch<32>(A, HW, n_tiles, s);
    case 64: return launch<64>(A, HW, n_tiles, s);
    case 128: return launch<128>(A, HW, n_tiles, s);
    default: return launch<256>(A, HW, n_tiles, s);
  }
}
