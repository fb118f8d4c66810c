// Attention of one new token per sequence over a paged KV cache, for gfx950, whose rows are
// bf16 or hold codes of 8 or 4 bits (mx.h), and whose sequences may begin alike.
//
//   o[b, h] = sum_j softmax_j(scale q[b, h] . k_j) v_j,   j < lens[b],
//
// k_j / v_j the rows of pool slot table[b][j / page] * page + j % page, query head h on
// kv head h / G.
//
// A sequence of n keys is cut into splits of split_keys(n) keys, a function of n alone, so
// a sequence's result does not depend on the rest of the batch nor on where its pages lie.
// The lengths are known on the device only: as many workgroups as are resident at once list
// the items there are and take them in turn, each requesting the first tile of its next one
// before it joins the waves of the present one.  (A grid over every split that the table has room
// for, most of which end at once: 218 us instead of 60 for 64 sequences of up to 8000 keys.)  An
// item is a split for one kv head, or a sequence of at most a tile's keys for four, one a wave.
// A second launch joins a sequence's splits, where the table has room for more than one.
//
// The four waves of a workgroup take the split's 32-key tiles in turn.  Scores are
// S^T = K Q^T by v_mfma_f32_16x16x32_bf16 with the G heads of the group in the 16 columns
// (the unused ones are zero); each lane then holds four keys of one head, the softmax runs
// there in fp32 with a lazily moved reference maximum, and the probabilities are used in
// place as the B operand of O^T += V^T P^T, as two bf16 terms: p cut to bf16 and the rest
// rounded to it (2^-15 of p is lost at most; the second product costs nothing next to the
// memory traffic).  Both terms are positive, so that an infinite v gives no inf - inf.  V
// goes from registers through a wave-private LDS stage to be read transposed.  Codes become
// bf16 in registers, exactly.  (The products that take codes and their scales as they are would
// save the conversions of K, but lose up to 2^-12 of the sum of their terms' sizes.)
//
// What bounds it: the K/V bytes, read once, where there are enough of them, and over 4-bit rows the
// instructions that a wave spends on a tile.  32 / 8 heads of 128, the same lengths in each format:
//   140161 keys, 131072 of them in one of six sequences: 574 MB of bf16 in 106 us (5.4 TB/s), 296 MB
//   of mxfp8 in 51 (5.8), 152 MB of mxfp4 in 36 (4.2; one wave per SIMD, splits as long as bf16's: 46)
//   54237 keys of 64 sequences of up to 8000: 222 MB in 43 us, 115 MB in 31, 59 MB in 27
// Below that the chain of dependent reads -- lengths, table, K/V, the second launch's partial sums
// (10 + 4 us for one sequence of 4097, whose 17 MB of bf16 take 3.3 of them).  With an earlier form
// over bf16: splits of 128 keys, 67 us instead of 64 for 64 sequences of up to 8000; of 512, 17
// instead of 13 for the one of 4097; at most 64 splits, or two tiles per wave requested at once: no
// difference.
//
// Keys that sequences of a batch share (prefix_rows, below) are split by their number alone, so that
// who shares them does not matter either; their splits are joined with the sequence's own.
#include <algorithm>

#include "keys64.h"
#include "mx.h"
#include "respect_amd.h"

namespace rspx {

namespace {

constexpr int kTile = 32;            // keys of a wave's step
constexpr int kWaves = 4;
constexpr int kSplitKeys = 256;      // the shortest split
// A longer cache gets longer splits.  Rows of few bits are bound by the waves that take them
// before they are by their bytes: twice the splits (131072 keys in mxfp4: 36 us for 46).
constexpr int most_splits(int bits) { return bits < 16 ? 64 : 32; }
constexpr int kSeqs = 1024;          // sequences of a launch
constexpr int kCUs = 256;
constexpr float kTiny = 1.17549435e-38f;   // the smallest normal number

// Shared beginnings: multiples of kKeys keys, in splits of their own.
constexpr int kMaxPrefixSplits = 64;
constexpr int kPrefixRows = 32 * kWaves;   // rows (sequences by heads of a group) of a workgroup
constexpr int kTileInts = 8;               // first sequence, rows, first row, first split, splits, keys

// Keys per split of a sequence of n keys: a multiple of kSplitKeys.
template <int BITS>
__host__ __device__ __forceinline__ int split_keys(int n) {
  constexpr unsigned kMost = most_splits(BITS);
  const unsigned per = ((unsigned)n + kMost - 1) / kMost;
  return per <= kSplitKeys ? kSplitKeys : (int)((per + kSplitKeys - 1) / kSplitKeys * kSplitKeys);
}
template <int BITS>
__host__ __device__ __forceinline__ int split_count(int n) {
  const unsigned k = (unsigned)split_keys<BITS>(n);
  return (int)(((unsigned)n + k - 1) / k);
}
// The most splits that any length up to n gives.
__host__ __forceinline__ int split_bound(int64_t n, int bits) {
  const int most = most_splits(bits);
  return n >= (int64_t)kSplitKeys * most ? most : (int)((n + kSplitKeys - 1) / kSplitKeys);
}

// The same for n shared keys: 20 splits of 128 to 512 keys, past that up to 64.
__host__ __device__ __forceinline__ int prefix_split_keys(int n) {
  auto parts = [&](unsigned m) { return ((unsigned)n + m * kKeys - 1) / (m * kKeys) * kKeys; };
  const unsigned per = parts(20);
  return per <= 128 ? 128 : per <= 512 ? (int)per : parts(64) <= 512 ? 512 : (int)parts(64);
}
__host__ __device__ __forceinline__ int prefix_splits(int n) {
  const unsigned k = (unsigned)prefix_split_keys(n);
  return (int)(((unsigned)n + k - 1) / k);
}
// The most splits that any n up to this one gives.
__host__ __forceinline__ int prefix_split_bound(int n) {
  const unsigned some = ((unsigned)n + 127) / 128, many = ((unsigned)n + 511) / 512;
  return (int)std::min<unsigned>(kMaxPrefixSplits, std::max<unsigned>(std::min<unsigned>(some, 20), many));
}

struct PagedArgs {
  const uint16_t* q;
  const char *k, *v;           // pools, strides in bytes
  const uint8_t *ks, *vs;      // their scales
  const int *table, *lens;
  const int *prefix, *tiles;   // keys that a sequence shares; what to compute of them
  uint16_t* out;
  float* po;                   // [B][H][smax][D]: a split's sums, the shared keys' splits first
  f32x2* pml;                  // [B][H][smax]: its m and l
  int64_t sqb, sqh, skh, skn, svh, svn, sksh, sksn, svsh, svsn, stb, sob, soh;
  int B, HK, G, pages, shift, width, smax, n_tiles, longest;
  float c;                     // scale * log2(e)
};

// Of a sequence of n keys that says it shares p: those that the launch's tiles compute, 0 where it
// is too short for them and goes through all of its own.
__device__ __forceinline__ int shared_keys(const PagedArgs& A, int p, int n) {
  return p > 0 && p <= A.longest && p <= n && n <= ((int64_t)A.width << A.shift) ? p : 0;
}

// A sequence of n > 0 keys as items, one for each workgroup that takes part: every split for every
// kv head, or, of no more keys than a wave takes at once, four kv heads (the result is the one that
// a workgroup's other waves, without keys, would leave as it is).
template <int BITS>
__device__ __forceinline__ int item_count(int n, int HK) {
  return n <= kTile ? (n > 0 ? (HK + kWaves - 1) / kWaves : 0) : split_count<BITS>(n) * HK;
}

// first[b]: the items of sequences before b (one for each kv head of a sequence without keys,
// whose rows are written too), length[b]: lens[b]; returns their number.  All 256 threads call it.
// The keys that from[b] says are shared are items elsewhere.
template <int BITS, bool SHARED>
__device__ __forceinline__ int list_items(const PagedArgs& A, int64_t cap, int* first, int* length, int* from) {
  const int* lens = A.lens;
  const int B = A.B;
  __shared__ int waves[4];
  constexpr int kPer = kSeqs / 256;
  // All loads before the first use: one after the other, 64 sequences in groups took 1.4 us longer.
  int cnt[kPer], lens_of[kPer], prefix_of[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = min((int)threadIdx.x * kPer + i, B - 1);
    lens_of[i] = lens[b];
    prefix_of[i] = SHARED ? A.prefix[b] : 0;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = threadIdx.x * kPer + i, n = lens_of[i];
    const int p = SHARED ? shared_keys(A, prefix_of[i], n) : 0;
    cnt[i] = b >= B ? 0 : n <= 0 || n > cap ? A.HK : item_count<BITS>(n - p, A.HK);
    sum += cnt[i];
    length[b] = n;
    if constexpr (SHARED) from[b] = p;
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

// The sequence that item i belongs to: the last one with first[b] <= i, by the counts of
// those up to i among every 16th and then among 16 (two reads of LDS one after the other, where a
// binary search makes ten).
__device__ __forceinline__ int find_seq(const int* first, int i) {
  static_assert(kSeqs == 64 * 16, "a lane holds 16");
  const int lane = threadIdx.x & 63;
  const int b = 16 * (__builtin_popcountll(__builtin_amdgcn_ballot_w64(first[16 * lane] <= i)) - 1);
  return b + __builtin_popcountll(__builtin_amdgcn_ballot_w64(first[b + (lane & 15)] <= i)) / 4 - 1;
}

// 16-byte unit swizzle of a staged V row: four consecutive keys' pairs of units lie in
// different banks for the transposing reads.
template <int D>
__device__ __forceinline__ int tile_vswizzle(int key) {
  constexpr int U = D / 8;
  if constexpr (U >= 16) return 2 * (key % 8);
  else return 2 * ((key / (16 / U)) % (U / 2));
}

// The byte offset of a row; the products of 64 bits are for strides of 4 GB and more, which the
// newer calls refuse.
template <bool WIDE>
__device__ __forceinline__ int64_t row_at(int row, int64_t stride) {
  return WIDE ? row * stride : (int64_t)((uint64_t)(uint32_t)row * (uint32_t)stride);
}

__device__ __forceinline__ float max4(float x) { return fmaxf(fmaxf(x, shfl_xor(x, 16)), fmaxf(shfl_xor(x, 32), shfl_xor(x, 48))); }
__device__ __forceinline__ float sum4(float x) {
  x = x + shfl_xor(x, 16);
  return x + shfl_xor(x, 32);
}

// Workgroups resident on a CU, by registers and LDS.
template <int D, int BITS>
struct PagedGeom {
  static constexpr int kPerCU = BITS < 16 ? (D >= 256 ? (BITS == 8 ? 1 : 2) : D >= 128 ? 3 : 4) : D >= 256 ? 1 : D >= 128 ? 2 : D >= 64 ? 3 : 4;
  static constexpr int kSharedPerCU = D >= 256 ? 1 : D >= 128 ? 2 : 3;
};

// One split of one sequence for one kv head.
struct Item {
  int g, b, from, n, split, splits;   // keys from .. from + n - 1
  int heads;                   // kv heads of the workgroup: this one, or one per wave
  int t, tend;                 // this wave's first tile, and the end of the split's
};

template <int D, bool SHARED>
struct PagedLds {
  char stage[kWaves][kTile * D * 2];
  float sm[kWaves][16], sl[kWaves][16];
  int first[kSeqs + 1], length[kSeqs], from[SHARED ? kSeqs : 1];
};

// Workgroup `block` of `blocks`: splits of the sequences' own keys.
template <int D, int BITS, bool SHARED>
__device__ __forceinline__ void paged_items(const PagedArgs& A, int block, int blocks, char (*stage)[kTile * D * 2],
                                            float (*sm)[16], float (*sl)[16], int* first, int* length, int* from) {
  constexpr int NQ = D / 32, DT = D / 16, U = D / 8;
  constexpr int RB = D * BITS / 8;                         // bytes of a row
  // K: lane (key, r4) takes KN loads of KW bytes, KF operands each; V: a tile is VL loads of VW
  // bytes per lane, VF units of the stage each.
  constexpr int KW = RB / 4 < 16 ? RB / 4 : 16, KN = RB / 4 / KW, KE = KW * 8 / BITS, KF = KE / 8;
  constexpr int VW = RB / 2 < 16 ? RB / 2 : 16, VU = RB / VW, VL = kTile * VU / 64, VE = VW * 8 / BITS, VF = VE / 8;

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, c16 = lane & 15, r4 = lane >> 4;
  const int64_t cap = (int64_t)A.width << A.shift;
  const int items = list_items<BITS, SHARED>(A, cap, first, length, from);
  if (block >= items) return;

  auto decode = [&](int i) {
    Item x;
    x.b = find_seq(first, i);
    const int r = i - __builtin_amdgcn_readfirstlane(first[x.b]);
    x.n = __builtin_amdgcn_readfirstlane(length[x.b]);
    x.g = r;
    x.split = x.splits = x.t = x.tend = x.from = 0;
    x.heads = 1;
    if (x.n > 0 && x.n <= cap) {
      if constexpr (SHARED) {
        x.from = __builtin_amdgcn_readfirstlane(from[x.b]);
        x.n -= x.from;
      }
      x.splits = split_count<BITS>(x.n);
      if (x.n <= kTile) {
        x.heads = kWaves;
        x.g = min(kWaves * r + w, A.HK - 1);
        x.tend = kWaves * r + w < A.HK;
      } else {
        const int per = split_keys<BITS>(x.n);
        x.split = r / A.HK;
        x.g = r - x.split * A.HK;
        x.t = x.split * (per / kTile) + w;
        x.tend = ((int)min((int64_t)x.n, (int64_t)(x.split + 1) * per) + kTile - 1) / kTile;
      }
    }
    return x;
  };
  // Key 32 t + lane % 32 (past the end: the last one): its page as the table has it, and its pool
  // slot, once that has come.  -1: the page is none, and nothing of it is read; or the wave has no
  // tile t.  No branch around the load: past one, all loads in flight would be waited for.
  auto page_of = [&](const Item& x, int t) {
    const bool on = t < x.tend;
    const int* row = on ? A.table + x.b * A.stb : A.lens;
    return row[on ? (x.from + min(t * kTile + (lane & 31), x.n - 1)) >> A.shift : 0];
  };
  auto slot_of = [&](const Item& x, int t, int p) {
    const int key = x.from + min(t * kTile + (lane & 31), x.n - 1);
    return t < x.tend && (unsigned)p < (unsigned)A.pages ? (p << A.shift) + (key & ((1 << A.shift) - 1)) : -1;
  };
  auto at = [&](int row, int64_t stride) { return row_at<BITS == 16 && !SHARED>(row, stride); };
  Words<KW> kf[2][KN];
  Words<VW> vf[VL];
  // Scales by the word (of a shorter row: all of them).  As bytes the compiler extends them where
  // paths meet, behind a wait for loads that have just begun.
  constexpr int KS = D >= 128 ? D / 128 : 1;
  uint32_t kscale[2][KS], vscale[VL];
  const int kfirst = KE * r4 / kGroup, vfirst = VE * (lane % VU) / kGroup;
  auto kscale_of = [&](int j, int i) {                     // of load i: KE elements from 4 KE i + KE r4 on
    return BITS < 16 ? scale_in(kscale[j][D >= 128 ? KE * i / kGroup : 0], kfirst + 4 * KE * i / kGroup) : 0.f;
  };
  auto vscale_of = [&](int j) { return BITS < 16 ? scale_in(vscale[j], vfirst) : 0.f; };
  auto load = [&](int g, int slot) {
    slot = max(slot, 0);
    const char* kb = A.k + g * A.skh;
    const char* vb = A.v + g * A.svh;
    const uint8_t *ks = A.ks + g * A.sksh, *vs = A.vs + g * A.svsh;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = shfl_idx_i(slot, 16 * j + c16);
      const char* p = kb + at(row, A.skn) + KW * r4;
#pragma unroll
      for (int i = 0; i < KN; ++i) kf[j][i] = load_words<KW>(p + 4 * KW * i);
      if constexpr (BITS < 16) {
#pragma unroll
        for (int i = 0; i < KS; ++i) kscale[j][i] = load_scales<D>(ks + at(row, A.sksn) + 4 * i);
      }
    }
#pragma unroll
    for (int j = 0; j < VL; ++j) {
      const int u = 64 * j + lane, row = shfl_idx_i(slot, u / VU);
      vf[j] = load_words<VW>(vb + at(row, A.svn) + VW * (u % VU));
      if constexpr (BITS < 16) vscale[j] = load_scales<D>(vs + at(row, A.svsn) + vfirst / 4 * 4);
    }
  };
  // B operand of the scores: lane (c16, r4) holds head c16, the head_dims of the lane's keys.
  bf16x8 qf[NQ];
  auto load_q = [&](const Item& x) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      u32x4 y = {0, 0, 0, 0};
      if (c16 < A.G)
        y = *reinterpret_cast<const u32x4*>(A.q + x.b * A.sqb + (int64_t)(x.g * A.G + c16) * A.sqh + KE * (4 * (i / KF) + r4) + 8 * (i % KF));
      qf[i] = __builtin_bit_cast(bf16x8, y);
    }
  };

  lds_char* st = (lds_char*)stage[w];
  Item cur = decode(block);
  const int page = page_of(cur, cur.t);
  load_q(cur);
  int slot = slot_of(cur, cur.t, page);                    // of the tile in kf and vf
  load(cur.g, slot);
  for (int item = block;;) {
    const int after = item + blocks;
    Item nxt = cur;
    nxt.t = nxt.tend = 0;
    if (after < items) nxt = decode(after);
    const int npage = page_of(nxt, nxt.t);
    int ahead = page_of(cur, cur.t + kWaves);              // the page of this item's next tile
    uint16_t* orow = A.out + cur.b * A.sob + (int64_t)cur.g * A.G * A.soh;

    float mref = kNone, lsum = 0.f;
    f32x4 acc[DT];
#pragma unroll
    for (int j = 0; j < DT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    bool bad = cur.t < cur.tend && slot < 0;
    if (cur.t >= cur.tend) {
      slot = slot_of(nxt, nxt.t, npage);
      load(nxt.g, slot);
    }
    for (int t = cur.t; t < cur.tend; t += kWaves) {
      f32x4 s[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NQ; ++i)
          s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
              __builtin_bit_cast(bf16x8, eight<BITS>(kf[j][i / KF], i % KF, kscale_of(j, i / KF))), qf[i], s[j], 0, 0, 0);
      }
      const int left = cur.n - t * kTile;                  // keys of the tile that exist
      if (left < kTile) {   // the repeated last row: its p of 0 times inf would be NaN
#pragma unroll
        for (int j = 0; j < VL; ++j)
          if ((64 * j + lane) / VU >= left) vf[j] = Words<VW>{}, vscale[j] = 0x01010101u * kLeastScale;
      }
      // The stage belongs to this wave, whose LDS operations keep their order: the reads of
      // the tile before are done before these writes land.
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const int u = 64 * j + lane, key = u / VU;
#pragma unroll
        for (int i = 0; i < VF; ++i)
          *(__attribute__((address_space(3))) u32x4*)(st + 16 * (key * U + ((u % VU * VF + i) ^ tile_vswizzle<D>(key)))) =
              eight<BITS>(vf[j], i, vscale_of(j));
      }
      // The next tile, of this item or the first of the next one.  Always some loads (row 0's where
      // there is none): the compiler counts those in flight the same on every path.
      const bool more = t + kWaves < cur.tend;
      int other = npage;
      asm volatile("" : "+v"(other));    // waited for here, not ahead of the loop
      const int mine = slot_of(cur, t + kWaves, ahead);
      bad |= more && mine < 0;
      slot = more ? mine : slot_of(nxt, nxt.t, other);
      ahead = page_of(cur, t + 2 * kWaves);
      load(more ? cur.g : nxt.g, slot);

      // Lane (c16, r4): head c16, keys 16 j + 4 r4 + e of the tile.
      float x[8], mx = kNegInf;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = s[i / 4][i % 4];
      }
      if (left < kTile) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (16 * (i / 4) + 4 * r4 + i % 4 >= left) x[i] = kNegInf;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, x[i]);
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
          h[z] = tr_read(st + 16 * (key * U + (u ^ tile_vswizzle<D>(key))) + 8 * (c16 & 1));
        }
        const bf16x8 va = __builtin_bit_cast(bf16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, ph, acc[j], 0, 0, 0);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pl, acc[j], 0, 0, 0);
      }
    }
    load_q(nxt);              // on its way while this item's waves are joined
    if (cur.splits == 0) {    // no keys: zeros; a length that does not fit: NaN
      for (int i = threadIdx.x; i < A.G * D; i += 256) orow[(i / D) * A.soh + i % D] = cur.n == 0 ? 0 : 0x7fc0;
    } else {
      if (__builtin_amdgcn_ballot_w64(bad) != 0) lsum = __builtin_nanf("");
      lsum = sum4(lsum);
      // The four waves' results, joined in wave order, or this wave's own.  A wave's stage holds its
      // [16][D] sums (the tile's V has been read by this wave).
      float* so = reinterpret_cast<float*>(&stage[0][0]);
#pragma unroll
      for (int j = 0; j < DT; ++j) *reinterpret_cast<f32x4*>(so + (w * 16 + c16) * D + (16 * j + 4 * r4)) = acc[j];
      if (r4 == 0) {
        sm[w][c16] = mref;
        sl[w][c16] = lsum;
      }
      const bool joined = cur.heads == 1;
      if (joined) lds_barrier();
      else asm volatile("" ::: "memory");   // a wave's LDS operations keep their order
      const int count = joined || cur.tend > 0 ? A.G * D : 0, stride = joined ? 256 : 64;
      for (int i = joined ? (int)threadIdx.x : lane; i < count; i += stride) {
        const int h = i / D, d = i % D;
        float m, o = 0.f, l = 0.f;
        if (joined) {
          m = sm[0][h];
#pragma unroll
          for (int k = 1; k < kWaves; ++k) m = fmaxf(m, sm[k][h]);
#pragma unroll
          for (int k = 0; k < kWaves; ++k) {
            const float a = fexp2(sm[k][h] - m);
            l = __builtin_fmaf(sl[k][h], a, l);
            o = __builtin_fmaf(so[(k * 16 + h) * D + d], a, o);
          }
        } else {
          m = sm[w][h], l = sl[w][h], o = o + so[(w * 16 + h) * D + d];   // as joined: no -0
        }
        if (cur.splits == 1 && cur.from == 0) {
          orow[h * A.soh + d] = f32_to_bf16_rne(o / l);
        } else {
          const int64_t p = (((int64_t)cur.b * A.HK + cur.g) * A.G + h) * A.smax + (SHARED ? prefix_splits(cur.from) : 0) + cur.split;
          A.po[p * D + d] = o;
          if (d == 0) A.pml[p] = f32x2{m, l};
        }
      }
      if (joined) lds_barrier();   // the stages and the waves' m and l have been read
    }
    if (after >= items) break;
    item = after;
    cur = nxt;
  }
}

// What bounds shared keys: for few rows the serial chain of a launch and a split's steps (4
// sequences behind 2496 keys: 11 us, 6 of them without any step); for many the partial sums, 520 bytes
// per row and split, and the steps (64 behind 8000 keys of bf16, 54 MB: 30 us, 8 of them the sums'
// 20 MB, where every sequence by itself would read 2.1 GB); for long ones the issue of a step's
// instructions and its chain LDS -> scores -> exponentials -> products (24 behind 100032 keys of
// mxfp4: 73 us, 0.54 PFLOP/s; without the products, staging alone 33).  20 splits up to 10240 keys:
// with 32, 34 us for the 64 and 8.4 instead of 7.1 to join them; with 16, 13 for the 4.  Steps of 64
// keys, one in flight: 168 us for the 24.
//
// What a tile says of shared keys: up to kPrefixRows rows (sequence b0 + r / G, head r % G of kv
// head g) and up to 4 / WR splits of the keys they share.  A wave takes 32 rows through one split,
// 32 keys a step; WR waves of different rows take the same split, and fetch its K and V together.
// What a wave computes of a row does not depend on WR, nor on the rows beside it.  The pages are those
// of the tile's first sequence that has all the shared keys.
//
// K and V come through registers, PF steps ahead, where they become bf16, into LDS: where waves
// share a split, into one of two slots while the other one is read, with one barrier a step.
// S^T = K Q^T by v_mfma_f32_32x32x16_bf16 leaves a row's scores in one lane and its neighbour of
// the other half; the probabilities, rounded to bf16 (half a step each) and summed as rounded, are
// used in place.  Every row sees all keys: there is no mask.  One term of p, as prompt attention has,
// and not the two of the sequences' own keys, since here products bound: with two, errors are those of
// a call without shared keys (0.0017 of the result's norm instead of 0.0023), and the 24 rows' 73 us become 94,
// the 64's 30 become 35, the 4's 10.5 become 11.6.
template <int D, int BITS, int WR>
__device__ __forceinline__ void prefix_rows(const PagedArgs& A, int total, const int (&T)[kTileInts], int g, char* lds) {
  constexpr int U = D / 8, NS = D / 16, DT = D / 32;
  // Bytes of a row and of a load, eight elements or more; loads of a row, of a step, of a thread.
  constexpr int kTeam = 64 * WR, RB = D * BITS / 8, kShare = kTile * RB / kTeam;
  constexpr int W = kShare >= 16 ? 16 : kShare > BITS ? kShare : BITS;
  constexpr int UR = RB / W, N = kTile * UR, UL = N > kTeam ? N / kTeam : 1;
  constexpr int E = W * 8 / BITS, EU = E / 8;
  // Steps in flight: as many as 64 registers hold (48 beside K operands read ahead; fewer where
  // more waves than two share a SIMD's).
  constexpr int kSet = UL * (W / 2 + (BITS < 16 ? 2 : 0)), kRoom = (D < 128 ? 32 : WR == 1 ? 64 : 48) / kSet;
  constexpr int PF = kRoom < 1 ? 1 : kRoom > 4 ? 4 : kRoom;
  constexpr int NB = WR == 1 ? 1 : 2, kBytes = kTile * D * 2;                    // K or V of a step in LDS
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5, tid = threadIdx.x % kTeam, team = w / WR;
  const int b0 = T[0], row0 = T[2], P = T[5], per = prefix_split_keys(P);
  const int rows = (int)min((int64_t)T[1], (int64_t)(total - b0) * A.G - row0) - 32 * (w % WR);   // from this wave's first on
  const int split = T[3] + team, key0 = team < T[4] ? split * per : 0;
  const int steps = team < T[4] ? (min(P - key0, per)) / kTile : 0;
  const int n = WR == 1 ? steps : (min(P - T[3] * per, per)) / kTile;            // the workgroup's longest
  if (WR == 1 && steps == 0) return;
  const bool active = rows > 0;
  // The first sequence of the tile that has all P keys names their pages: a shorter one's row may hold
  // anything behind its end.  Those of the tile's first one are requested beside the lengths.
  int lead = b0 + row0 / A.G;
  const int many = rows + 32 * (w % WR);
  auto has = [&](int r) { return shared_keys(A, P, A.lens[b0 + (row0 + min(r, many - 1)) / A.G]) > 0 && r < many; };
  const bool has_lo = has(lane), has_hi = WR == 4 && has(lane + 64);
  const int row = row0 + 32 * (w % WR) + min(col, max(rows - 1, 0));
  const int b = b0 + (active ? row / A.G : 0), h = g * A.G + (active ? row % A.G : 0);
  const int keys = A.lens[b], prefix = A.prefix[b];

  // B operand of the scores: lane (col, half) holds row col, head_dim 16 i + 8 half .. + 7.
  bf16x8 qf[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i)
    qf[i] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(A.q + b * A.sqb + (int64_t)h * A.sqh + 8 * half + 16 * i));

  // The page of key 32 t + lane % 32 of the split (of a step there is not: of the last one's), and
  // its slot, once that has come (0 where there is none).
  const int* table = A.table + (int64_t)lead * A.stb;
  bool bad = false;
  auto key_of = [&](int t) { return (steps > 0 ? key0 + kTile * min(t, steps - 1) : 0) + (lane & 31); };
  auto page_of = [&](int t) { return table[key_of(t) >> A.shift]; };
  auto slot_of = [&](int t, int p) {
    const bool ok = (unsigned)p < (unsigned)A.pages;
    bad |= t < steps && !ok;
    return ok && t < steps ? (p << A.shift) + (key_of(t) & ((1 << A.shift) - 1)) : 0;
  };

  // Load j of this thread: bytes W c of key u / UR, u = kTeam j + tid, of K and of V.
  Words<W> rk[PF][UL], rv[PF][UL];
  uint32_t sk[PF][UL], sv[PF][UL];
  const int c = tid % UR, scale = E * c / kGroup;
  const char *kb = A.k + g * A.skh + W * c, *vb = A.v + g * A.svh + W * c;
  const uint8_t *ksb = A.ks + g * A.sksh + scale / 4 * 4, *vsb = A.vs + g * A.svsh + scale / 4 * 4;
  struct RowsOf {
    int r[UL];
  };
  auto rows_of = [&](int slot) {
    RowsOf x;
#pragma unroll
    for (int j = 0; j < UL; ++j) x.r[j] = shfl_idx_i(slot, (kTeam * j + tid) % N / UR);
    return x;
  };
  auto fetch = [&](int set, const RowsOf& x) {
#pragma unroll
    for (int j = 0; j < UL; ++j) {
      const int r = x.r[j];
      rk[set][j] = load_words<W>(kb + row_at<false>(r, A.skn));
      rv[set][j] = load_words<W>(vb + row_at<false>(r, A.svn));
      if constexpr (BITS < 16) {
        sk[set][j] = load_scales<D>(ksb + row_at<false>(r, A.sksn));
        sv[set][j] = load_scales<D>(vsb + row_at<false>(r, A.svsn));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  lds_char* base = (lds_char*)lds + team * (NB * 2 * kBytes);
  auto put = [&](int set, int slot) {
#pragma unroll
    for (int j = 0; j < UL; ++j) {
      const int key = (kTeam * j + tid) % N / UR;
      const float fk = BITS < 16 ? scale_in(sk[set][j], scale) : 0.f, fv = BITS < 16 ? scale_in(sv[set][j], scale) : 0.f;
#pragma unroll
      for (int i = 0; i < EU; ++i) {
        const int u = c * EU + i;
        lds_char* d = base + 2 * kBytes * slot + 16 * key * U;
        *(__attribute__((address_space(3))) u32x4*)(d + 16 * (u ^ kswizzle<D>(key))) = eight<BITS>(rk[set][j], i, fk);
        *(__attribute__((address_space(3))) u32x4*)(d + kBytes + 16 * (u ^ vswizzle<D>(key))) = eight<BITS>(rv[set][j], i, fv);
      }
    }
  };

  int k_at = 16 * (col * U + (half ^ kswizzle<D>(col)));
  int v_at;
  {
    const int l16 = lane & 15, key = 4 * half + (l16 >> 2), u = 2 * ((lane >> 4) & 1) + ((l16 & 3) >> 1);
    v_at = 16 * (key * U + (u ^ vswizzle<D>(key))) + 8 * (l16 & 1);
  }
  asm("" : "+v"(k_at), "+v"(v_at));

  float mref = kNone, lsum = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int j = 0; j < DT; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;
  u32x4 kf[NS];                                            // A operands of the scores
  auto read_k = [&](int slot) {
#pragma unroll
    for (int i = 0; i < NS; ++i) kf[i] = read16(base + 2 * kBytes * slot + (k_at ^ (32 * i)));
  };
  auto compute = [&](int slot) {
    const lds_char* dv = base + 2 * kBytes * slot + kBytes;
    // Lane (col, half): row col, keys 8 (e / 4) + 4 half + e % 4.
    f32x16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kf[i]), qf[i], s, 0, 0, 0);
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
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
    u32x4 p[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = fexp2(__builtin_fmaf(s[2 * i], A.c, -mref)), y = fexp2(__builtin_fmaf(s[2 * i + 1], A.c, -mref));
      p[i / 4][i % 4] = pack_bf16x2(x, y);
      lsum = dot2(p[i / 4][i % 4], lsum);
    }
    // A operand of head_dim tile j, 16-key step i: V[key][32 j + lane % 32], k-slots
    // 8 half + e <-> keys 16 i + 8 (e / 4) + 4 half + e % 4, the order in which the lane holds p.
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        s16x4 h[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) h[z] = tr_read(dv + (v_at ^ (64 * j)) + 16 * U * (16 * i + 8 * z));
        acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7)),
            __builtin_bit_cast(bf16x8, p[i]), acc[j], 0, 0, 0);
      }
  };

  // No branch around the loads: past one, all in flight would be waited for.
  int page[PF];
#pragma unroll
  for (int i = 0; i < PF; ++i) page[i] = page_of(i);
  {
    const uint64_t lo = __builtin_amdgcn_ballot_w64(has_lo), hi = __builtin_amdgcn_ballot_w64(has_hi);
    if ((lo | hi) == 0) return;                            // no row of the tile takes part
    const int other = b0 + (row0 + (lo ? __builtin_ctzll(lo) : 64 + __builtin_ctzll(hi))) / A.G;
    if (other != lead) {
      table = A.table + (int64_t)(lead = other) * A.stb;
#pragma unroll
      for (int i = 0; i < PF; ++i) page[i] = page_of(i);
    }
  }
  auto next = [&](int set, int t) {
    const RowsOf x = rows_of(slot_of(t, page[set]));
    page[set] = page_of(t + PF);
    fetch(set, x);
  };
#pragma unroll
  for (int i = 0; i < PF; ++i) next(i, i);
  if constexpr (NB == 2) {
    put(0, 0);
    next(0, PF);
    lds_barrier();                                         // step 0 is in place
  }
  for (int t0 = 0;; t0 += PF) {
#pragma unroll
    for (int i = 0; i < PF; ++i) {
      const int t = t0 + i, set = NB == 2 ? (i + 1) % PF : i, slot = NB == 2 ? t & 1 : 0, ahead = t + PF + (NB == 2);
      if constexpr (NB == 2) read_k(slot);
      const RowsOf x = rows_of(slot_of(ahead, page[set]));
      page[set] = page_of(ahead + PF);
      put(set, NB == 2 ? slot ^ 1 : 0);                    // step t + 1, where step t - 1 has been read; or step t
      fetch(set, x);
      asm volatile("" ::: "memory");
      if constexpr (NB == 1) read_k(0);
      if (active && t < steps) compute(slot);
      if constexpr (NB == 2) lds_barrier();
      if (t + 1 >= n) goto done;
    }
  }
done:
  // A page that is none spoils every row that reads it.
  lsum = lsum + shfl_xor(lsum, 32);
  if (__builtin_amdgcn_ballot_w64(bad) != 0) lsum = __builtin_nanf("");
  // A sequence that goes through all of its keys by itself has its own splits where these would be.
  if (col >= rows || steps == 0 || shared_keys(A, prefix, keys) == 0) return;
  const int64_t at = ((int64_t)b * A.HK * A.G + h) * A.smax + split;
#pragma unroll
  for (int j = 0; j < DT; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<f32x4*>(A.po + at * D + 32 * j + 8 * e + 4 * half) =
          f32x4{acc[j][4 * e], acc[j][4 * e + 1], acc[j][4 * e + 2], acc[j][4 * e + 3]};
  if (half == 0) A.pml[at] = f32x2{mref, lsum};
}

// Waves of a tile's rows: they share a split, the others take the next ones.
__host__ __device__ __forceinline__ int prefix_waves(int rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

template <int D, int BITS>
__device__ __forceinline__ void prefix_tile(const PagedArgs& A, int total, int index, char* lds) {
  const int g = index % A.HK;
  int T[kTileInts];
  __builtin_memcpy(T, A.tiles + (int64_t)(index / A.HK) * kTileInts, sizeof T);
#pragma unroll
  for (int i = 0; i < kTileInts; ++i) T[i] = __builtin_amdgcn_readfirstlane(T[i]);
  const int b0 = T[0], rows = T[1], row0 = T[2], split0 = T[3], splits = T[4], P = T[5];
  if (b0 < 0 || b0 >= total || rows < 1 || rows > kPrefixRows || row0 < 0 || row0 >= (int64_t)(total - b0) * A.G) return;
  if (P < kKeys || P % kKeys || P > A.longest || P > ((int64_t)A.width << A.shift)) return;
  if (split0 < 0 || splits < 1 || splits > 4 / prefix_waves(rows) || split0 > prefix_splits(P) - splits) return;
  if (rows <= 32) prefix_rows<D, BITS, 1>(A, total, T, g, lds);
  else if (rows <= 64) prefix_rows<D, BITS, 2>(A, total, T, g, lds);
  else prefix_rows<D, BITS, 4>(A, total, T, g, lds);
}

template <int D, int BITS>
__global__ __launch_bounds__(256, (PagedGeom<D, BITS>::kPerCU)) void paged_attn_kernel(PagedArgs A) {
  __shared__ __align__(16) char stage[kWaves][kTile * D * 2];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  __shared__ int first[kSeqs + 1], length[kSeqs];
  paged_items<D, BITS, false>(A, blockIdx.x, gridDim.x, stage, sm, sl, first, length, nullptr);
}

// The first `tiles` workgroups take the shared keys, the rest the sequences' own.
template <int D, int BITS>
__global__ __launch_bounds__(256, (PagedGeom<D, BITS>::kSharedPerCU)) void shared_attn_kernel(PagedArgs A, int total, int tiles) {
  constexpr int kPrefixBytes = 2 * kWaves * kTile * D * 2;
  __shared__ __align__(16) char lds[sizeof(PagedLds<D, true>) > kPrefixBytes ? sizeof(PagedLds<D, true>) : kPrefixBytes];
  if ((int)blockIdx.x < tiles) {
    prefix_tile<D, BITS>(A, total, blockIdx.x, lds);
  } else {
    auto& x = *reinterpret_cast<PagedLds<D, true>*>(lds);
    paged_items<D, BITS, true>(A, blockIdx.x - tiles, gridDim.x - tiles, x.stage, x.sm, x.sl, x.first, x.length, x.from);
  }
}

// One workgroup per (query head, sequence).  Every wave takes the splits' weights, lane s
// that of split s; then lanes of four columns each sum every (256 / (D / 4))-th split, and
// those sums are added in order.
template <int D, int BITS, bool SHARED>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs A) {
  constexpr int L = D / 4, P = 256 / L, kMost = most_splits(BITS) + (SHARED ? kMaxPrefixSplits : 0);
  constexpr int R = (kMost + 63) / 64;                     // splits of a lane: lane, lane + 64
  __shared__ float wt[64 * R];
  __shared__ __align__(16) f32x4 sums[P][L];
  const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63;
  const int64_t p = ((int64_t)b * A.HK * A.G + h) * A.smax;
  f32x2 ml[R];
#pragma unroll
  for (int i = 0; i < R; ++i) ml[i] = lane + 64 * i < A.smax ? A.pml[p + lane + 64 * i] : f32x2{kNone, 0.f};   // beside the length
  const int n = A.lens[b], prefix = SHARED ? A.prefix[b] : 0;
  if (n <= 0 || n > ((int64_t)A.width << A.shift)) return;
  const int from = SHARED ? shared_keys(A, prefix, n) : 0;
  const int splits = (from > 0 ? prefix_splits(from) : 0) + split_count<BITS>(n - from);
  if (splits == 1 && from == 0) return;
  const int c = threadIdx.x % L, part = threadIdx.x / L;
  constexpr int N = (kMost + P - 1) / P;
  f32x4 x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = part + P * i;
    x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s < splits) x[i] = *reinterpret_cast<const f32x4*>(A.po + (p + s) * D + 4 * c);
  }
  float m = kNone;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (lane + 64 * i >= splits) ml[i] = f32x2{kNone, 0.f};
    m = fmaxf(m, ml[i][0]);
  }
  for (int k = 32; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k));
  float l = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const float a = fexp2(ml[i][0] - m);
    l = i == 0 ? ml[i][1] * a : __builtin_fmaf(ml[i][1], a, l);
    if (threadIdx.x < 64) wt[lane + 64 * i] = a;
  }
  for (int k = 32; k >= 1; k >>= 1) l = l + __shfl_xor(l, k);
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

template <int D, int BITS, bool SHARED>
int launch(PagedArgs A, int B, hipStream_t s) {
  const int psmax = SHARED ? prefix_split_bound(A.longest) : 0;
  for (int b0 = 0; b0 < B; b0 += kSeqs) {
    A.B = B - b0 < kSeqs ? B - b0 : kSeqs;
    const int64_t items = (int64_t)A.B * (A.smax - psmax) * A.HK, most = kCUs * (SHARED ? PagedGeom<D, BITS>::kSharedPerCU : PagedGeom<D, BITS>::kPerCU);
    const unsigned blocks = (unsigned)(items < most ? items : most);
    if constexpr (SHARED) {
      const int tiles = b0 == 0 ? A.n_tiles * A.HK : 0;    // of all sequences
      hipLaunchKernelGGL((shared_attn_kernel<D, BITS>), dim3(tiles + blocks), dim3(256), 0, s, A, B, tiles);
    } else {
      hipLaunchKernelGGL((paged_attn_kernel<D, BITS>), dim3(blocks), dim3(256), 0, s, A);
    }
    if (A.smax > 1) hipLaunchKernelGGL((paged_join_kernel<D, BITS, SHARED>), dim3(A.HK * A.G, A.B), dim3(256), 0, s, A);
    A.q += A.B * A.sqb;
    A.out += A.B * A.sob;
    A.table += A.B * A.stb;
    A.lens += A.B;
    if constexpr (SHARED) A.prefix += A.B;
    A.po += (int64_t)A.B * A.HK * A.G * A.smax * D;
    A.pml += (int64_t)A.B * A.HK * A.G * A.smax;
  }
  return hipGetLastError() == hipSuccess ? RSPX_OK : RSPX_ELAUNCH;
}

template <int BITS, bool SHARED>
int launch_for(int D, const PagedArgs& A, int B, hipStream_t s) {
  switch (D) {
    case 32: return launch<32, BITS, SHARED>(A, B, s);
    case 64: return launch<64, BITS, SHARED>(A, B, s);
    case 128: return launch<128, BITS, SHARED>(A, B, s);
    default: return launch<256, BITS, SHARED>(A, B, s);
  }
}

bool head_dim_ok(int D) { return D == 32 || D == 64 || D == 128 || D == 256; }

int64_t workspace(int B, int H, int D, int page, int width, int psmax, int bits) {
  if (B < 0 || H < 1 || page < 1 || width < 0 || !head_dim_ok(D)) return -1;
  const int smax = split_bound((int64_t)width * page, bits) + psmax;
  return smax <= 1 ? 0 : (int64_t)B * H * smax * (D + 2) * 4;
}

// A pool as the C ABI names it: strides in its elements.
struct PoolArg {
  const void* rows;
  int64_t sh, sn;
  const void* scales;
  int64_t ssh, ssn;
};

int attend(const void* q, int64_t sqb, int64_t sqh, const PoolArg& k, const PoolArg& v, int bits, const int32_t* table,
           int64_t stb, const int32_t* lens, bool shared, const int32_t* prefix, const int32_t* tiles, int n_tiles, int longest,
           void* out, int64_t sob, int64_t soh, int B, int H, int HK, int D, int pages, int page, int width, float sm_scale,
           void* ws, int64_t ws_bytes, void* stream) {
  if (B < 0 || H < 1 || HK < 1 || H % HK || pages < 1 || page < 1 || (page & (page - 1)) || width < 0) return RSPX_EINVAL;
  if (!(sm_scale > 0.f) || sm_scale > 3e38f) return RSPX_EINVAL;
  if ((int64_t)pages * page > INT32_MAX || (int64_t)width * page > INT32_MAX - 4096) return RSPX_EINVAL;
  if (n_tiles < 0 || longest < 0 || longest > (int64_t)width * page) return RSPX_EINVAL;
  if (bits != 16 && bits != 8 && bits != 4) return RSPX_EUNSUPPORTED;
  if (!head_dim_ok(D) || H / HK > 16 || HK > 4096) return RSPX_EUNSUPPORTED;   // items of a launch are counted in 32 bits
  if ((int64_t)n_tiles * HK > (1 << 23)) return RSPX_EUNSUPPORTED;             // a grid dimension holds 2^32 threads
  if (B == 0) return RSPX_OK;
  if (!q || !k.rows || !v.rows || !lens || !out || (width && !table)) return RSPX_EINVAL;
  if (bits < 16 && (!k.scales || !v.scales)) return RSPX_EINVAL;
  if (bits < 16 || shared)
    for (const int64_t s : {k.sn, v.sn, bits < 16 ? k.ssn : 0, bits < 16 ? v.ssn : 0})
      if (s < 0 || s > INT32_MAX) return s < 0 ? RSPX_EINVAL : RSPX_EUNSUPPORTED;
  if (shared && (!prefix || (n_tiles && !tiles))) return RSPX_EINVAL;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  if (reinterpret_cast<uintptr_t>(out) & 1u) return RSPX_EALIGN;
  const int unit = bits == 16 ? 8 : 16;
  if (!al(q) || !al(k.rows) || !al(v.rows) || sqb % 8 || sqh % 8 || k.sh % unit || k.sn % unit || v.sh % unit || v.sn % unit)
    return RSPX_EALIGN;
  const int psmax = shared ? prefix_split_bound(longest) : 0;
  const int64_t need = workspace(B, H, D, page, width, psmax, bits);
  if (need > 0 && (!ws || ws_bytes < need)) return RSPX_EWORKSPACE;
  if (need > 0 && !al(ws)) return RSPX_EALIGN;
  const int64_t e = bits == 16 ? 2 : 1;
  PagedArgs A;
  A.q = static_cast<const uint16_t*>(q);
  A.k = static_cast<const char*>(k.rows);
  A.v = static_cast<const char*>(v.rows);
  A.ks = static_cast<const uint8_t*>(k.scales);
  A.vs = static_cast<const uint8_t*>(v.scales);
  A.table = table;
  A.lens = lens;
  A.prefix = prefix, A.tiles = tiles, A.n_tiles = n_tiles, A.longest = longest;
  A.out = static_cast<uint16_t*>(out);
  A.po = static_cast<float*>(ws);
  A.sqb = sqb, A.sqh = sqh, A.stb = stb, A.sob = sob, A.soh = soh;
  A.skh = k.sh * e, A.skn = k.sn * e, A.svh = v.sh * e, A.svn = v.sn * e;
  A.sksh = k.ssh, A.sksn = k.ssn, A.svsh = v.ssh, A.svsn = v.ssn;
  A.HK = HK, A.G = H / HK, A.pages = pages, A.width = width;
  A.shift = __builtin_ctz((unsigned)page);
  const int smax = split_bound((int64_t)width * page, bits);
  A.smax = (smax < 1 ? 1 : smax) + psmax;
  A.pml = reinterpret_cast<f32x2*>(A.po + (int64_t)B * H * A.smax * D);
  A.c = sm_scale * 1.44269504088896340736f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (shared) {
    if (bits == 16) return launch_for<16, true>(D, A, B, s);
    return bits == 8 ? launch_for<8, true>(D, A, B, s) : launch_for<4, true>(D, A, B, s);
  }
  if (bits == 16) return launch_for<16, false>(D, A, B, s);
  return bits == 8 ? launch_for<8, false>(D, A, B, s) : launch_for<4, false>(D, A, B, s);
}

}  // namespace

}  // namespace rspx

using namespace rspx;

extern "C" int64_t rspx_paged_attn_workspace_bytes(int B, int H, int D, int page, int width) {
  return workspace(B, H, D, page, width, 0, RSPX_BF16);
}

extern "C" int rspx_paged_attn(const void* q, int64_t sqb, int64_t sqh, const void* kc, int64_t skh, int64_t skn,
                               const void* vc, int64_t svh, int64_t svn, const int32_t* table, int64_t stb,
                               const int32_t* lens, void* out, int64_t sob, int64_t soh, int B, int H, int HK, int D,
                               int pages, int page, int width, float sm_scale, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  return attend(q, sqb, sqh, PoolArg{kc, skh, skn, nullptr, 0, 0}, PoolArg{vc, svh, svn, nullptr, 0, 0}, RSPX_BF16, table, stb,
                lens, false, nullptr, nullptr, 0, 0, out, sob, soh, B, H, HK, D, pages, page, width, sm_scale, workspace,
                workspace_bytes, stream);
}

extern "C" int rspx_paged_attn_mx(const void* q, int64_t sqb, int64_t sqh, const void* k_codes, int64_t skch, int64_t skcn,
                                  const void* k_scales, int64_t sksh, int64_t sksn, const void* v_codes, int64_t svch,
                                  int64_t svcn, const void* v_scales, int64_t svsh, int64_t svsn, const int32_t* table,
                                  int64_t stb, const int32_t* lens, void* out, int64_t sob, int64_t soh, int B, int H, int HK,
                                  int D, int pages, int page, int width, float sm_scale, int format, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (format == RSPX_BF16) return RSPX_EUNSUPPORTED;   // rspx_paged_attn
  return attend(q, sqb, sqh, PoolArg{k_codes, skch, skcn, k_scales, sksh, sksn}, PoolArg{v_codes, svch, svcn, v_scales, svsh, svsn},
                format, table, stb, lens, false, nullptr, nullptr, 0, 0, out, sob, soh, B, H, HK, D, pages, page, width, sm_scale,
                workspace, workspace_bytes, stream);
}

extern "C" int64_t rspx_shared_plan(const int64_t* members, const int64_t* keys, int n, int group, int32_t* prefix,
                                    int32_t* tiles) {
  if (n < 0 || group < 1 || group > 16 || (n > 0 && (!members || !keys))) return RSPX_EINVAL;
  int64_t b = 0, count = 0;
  for (int i = 0; i < n; ++i) {
    if (members[i] < 0 || keys[i] < 0 || members[i] > INT32_MAX || keys[i] > INT32_MAX) return RSPX_EINVAL;
    // One sequence alone shares nothing; a begun step is left to the sequences themselves.
    const int p = members[i] < 2 ? 0 : (int)(keys[i] / kKeys * kKeys);
    if (b + members[i] > INT32_MAX / 16) return RSPX_EINVAL;
    if (prefix) std::fill(prefix + b, prefix + b + members[i], p);
    const int rows = (int)members[i] * group, splits = p ? prefix_splits(p) : 0;
    // The row blocks of a split beside one another: they read the same keys.
    for (int split = 0; split < splits; split += 4)
      for (int64_t r = 0; r < rows; r += kPrefixRows) {    // past the last of 2^31 - 16 rows it is 2^31
        const int part = (int)std::min<int64_t>(rows - r, kPrefixRows), each = 4 / prefix_waves(part);
        for (int k = split; k < std::min(split + 4, splits); k += each, ++count)
          if (tiles) {
            int32_t* t = tiles + count * kTileInts;
            t[0] = (int32_t)b, t[1] = part, t[2] = (int32_t)r, t[3] = k, t[4] = std::min({each, splits - k, split + 4 - k});
            t[5] = p, t[6] = t[7] = 0;
          }
      }
    b += members[i];
  }
  return count;
}

extern "C" int64_t rspx_paged_attn_shared_workspace_bytes(int B, int H, int D, int page, int width, int longest, int format) {
  if (longest < 0 || (format != RSPX_BF16 && format != RSPX_MXFP8 && format != RSPX_MXFP4)) return -1;
  return workspace(B, H, D, page, width, prefix_split_bound(longest), format);
}

extern "C" int rspx_paged_attn_shared(const void* q, int64_t sqb, int64_t sqh, const void* kc, int64_t skh, int64_t skn,
                                      const void* k_scales, int64_t sksh, int64_t sksn, const void* vc, int64_t svh, int64_t svn,
                                      const void* v_scales, int64_t svsh, int64_t svsn, const int32_t* table, int64_t stb,
                                      const int32_t* lens, const int32_t* prefix, const int32_t* tiles, int n_tiles, int longest,
                                      void* out, int64_t sob, int64_t soh, int B, int H, int HK, int D, int pages, int page,
                                      int width, float sm_scale, int format, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
  return attend(q, sqb, sqh, PoolArg{kc, skh, skn, k_scales, sksh, sksn}, PoolArg{vc, svh, svn, v_scales, svsh, svsn}, format,
                table, stb, lens, true, prefix, tiles, n_tiles, longest, out, sob, soh, B, H, HK, D, pages, page, width, sm_scale,
                workspace, workspace_bytes, stream);
}
