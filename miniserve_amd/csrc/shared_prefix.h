// Attention for a batch whose rows come in groups, each group behind a prefix of its own: the
// same physical pages in every row of the group (gfx950; a bf16/fp16 query over a cache of its
// type or of fp8 e4m3, head_dim 64 or 128, one query token a row or several).
//
// The work is a list of segments: one a group (the prefix's keys, read once for the query rows of
// every member) and one a batch row (the keys past its prefix, or all of them). A segment falls
// into units, one a KV head and block of up to 128 query rows; a unit's keys are cut into tiles
// of 32 KB of K and 32 KB of V. All tiles of all units, in order, are dealt in equal contiguous
// shares, one a workgroup, whatever the lengths (they are read on the device, so a call is
// capture-safe). A share's part of one unit is a piece; it leaves, for each of its query rows,
//   m = max_j s_j,  l = sum_j 2^(s_j - m),  acc = sum_j 2^(s_j - m) V_j,   s_j = scale log2(e) q.K_j
// over the piece's visible keys, and the merge kernel below joins a row's pieces:
//   out = sum 2^(m - M) acc / sum 2^(m - M) l,   M = max m.
//
// Few query rows wait for the memory pipe, many for the matrix cores and the softmax (a tile of 128
// rows costs 2 to 4 times one of 8), so the shares are equal in cost, not in tiles (ShCost).
//
// A workgroup has four copying waves, one a SIMD, and eight computing ones. The copying waves bring
// the share's tiles into two LDS slots with the load unit, one tile ahead of the computation and on
// across pieces and units, so that the memory pipe does not run dry between them, and keep the page
// walk out of the computing waves. Those take 16 query rows each: scores are S^T = K Q^T on
// v_mfma_f32_16x16x32, so that lane (g, n) = (l / 16, l % 16) holds row n's scores of keys
// 4 g .. 4 g + 3 of a 16-key block, and two such blocks, rounded to the query type and packed, are
// its B operand of O^T += V^T P^T (V^T by transposed LDS reads): softmax and rescaling stay in the
// lane. A unit of 64 rows or fewer leaves computing waves over, which take other 32-key blocks of
// the same rows and are joined through LDS at the piece's end. (Four waves of 32 rows read K and V
// from LDS half as often, but one wave a SIMD does not hide the reads' and products' latencies:
// draft rows below 37.5 us against 32.9.)
//
// The kernel runs each part of its code a few times a workgroup, so its size counts: every part
// stands once, divisions by the call's constants are multiplications, and the plan's searches are
// made for 64 tiles at a time, a lane each.
//
// Measured (this launch, then the merge): 64 rows of H32/KVH8/D128 bf16 in 8 groups of 8, prefixes
// of 1024 to 8192 keys and 64 to 1024 own ones, 48 + 4.6 us (225 MB: 36 us of pure reading); 128
// rows over an fp8 cache behind one prefix of 8192, 94 + 5.9 us (259 MB, 19 GFLOP); 32 rows of 4
// draft tokens, H28/KVH4 fp16, in 4 groups, 30 + 6.0 us; 6 rows of a small model 11 + 3.9 us, of
// which the launch, the plan and the first tile's latency are nearly all. What bounds it: the plan
// and the first window, 9000 clocks a workgroup before the first copy; about 6000 a piece; between
// them the reads' rate for few rows and some 1300 clocks a 32-key block for 128 (1900 over fp8).
//
// Semantics: miniserve/attention.py:205-250 (causal), whose gather reads a shared page once a row.
#pragma once

#include "prefill_mfma.h"

namespace msattn {

constexpr int kShCopy = 4;              // copying waves: one a SIMD
constexpr int kShComp = 8;              // computing waves: two a SIMD
constexpr int kShThreads = 64 * (kShComp + kShCopy);
constexpr int kShRows = 16 * kShComp;   // query rows of a unit, at most: 16 a computing wave
constexpr int kShMaxBatch = 1024;       // rows (and groups) of a launch: its plan sits in LDS
constexpr int kShHalf = 32 * 1024;      // bytes of K, and of V, of a tile
constexpr int kShSlots = 2;             // tiles in LDS
// Keys of a tile.
__host__ __device__ constexpr int sh_tile(int head_dim, int kv_bytes) {
  return kShHalf / (head_dim * kv_bytes);
}
// Cache policy of the reads of a 16-bit cache in units whose keys no other row block reads (2:
// nontemporal; 64 rows in 8 groups of H32/KVH8/D128 48 us against 56, H16/KVH2/D64 28 and 29 with
// the merge). Keys that several row blocks read stay in L2 for them (nontemporal, 16 rows of 32
// query rows took 2 % more), and an fp8 cache's took 1 to 3 % more.
#ifndef MSATTN_SHARED_AUX
#define MSATTN_SHARED_AUX 2
#endif
constexpr int kShAux = MSATTN_SHARED_AUX;

// What a share is to cost a workgroup, in units of about 250 clocks: a piece (its query, its plan,
// its partials), and each 32-key block of a unit of so many rows. Few rows wait for the memory pipe,
// many for the matrix cores and the softmax. (From a fit of the workgroups' clocks to their pieces
// and blocks, then tried around. 64 rows in 8 groups of H32/KVH8/D128 took 81 us in shares of equal
// tiles, 63 with one row of costs for all types and sizes and 56 with these, all before the
// nontemporal reads. 40 calls of H14/KVH2/D64, H16/KVH8/D64, H28/KVH4/D128 and H32/KVH8/D128, 16-bit
// and fp8, 16 to 64 rows in 1 to 8 groups, 1 to 4 tokens: the first row for all 2 % less to 28 % more
// but for one call of 16 rows (H28/KVH4 over fp8, 18.4 us here, 15.1), block costs halved 2 % less to
// 26 % more, half as much again 6 % less to 9 % more but for the same call.)
#ifndef MSATTN_SHARED_COSTS
#define MSATTN_SHARED_COSTS {20, 6, 7, 9, 12}, {20, 3, 4, 5, 7}, {20, 2, 3, 5, 8}, {20, 2, 3, 4, 6}
#endif
template <int D, int EB>
struct ShCost {
  static constexpr int row(int i) {  // 16-bit caches of head_dim 128 and 64, fp8 ones
    constexpr int c[4][5] = {MSATTN_SHARED_COSTS};
    return c[(EB == 1 ? 2 : 0) + (D == 64 ? 1 : 0)][i];
  }
  static constexpr int kPiece = row(0);
  __device__ static int block(int rows) {
    constexpr int c[4] = {row(1), row(2), row(3), row(4)};
    return rows > 64 ? c[3] : (rows > 32 ? c[2] : (rows > 16 ? c[1] : c[0]));
  }
};

// Division of x < 2^31 by a constant of the call: with s = ceil(log2 d) and m = ceil(2^(31+s) / d),
// x m 2^-(31+s) exceeds x / d by less than 1 / d, so its integer part is the quotient.
struct FastDiv {
  uint32_t m;
  int s;
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f;
  f.s = 0;
  while ((uint32_t(1) << f.s) < d) ++f.s;
  f.m = static_cast<uint32_t>(((uint64_t(1) << (31 + f.s)) + d - 1) / d);
  return f;
}
__device__ __forceinline__ int fast_quot(int x, FastDiv f) {
  return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(x), f.m) >> f.s);
}

struct SharedParams {
  const void* q;
  const void* k;
  const void* v;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* group_rows;    // [groups + 1]
  const int32_t* prefix_pages;  // [groups]
  void* out;
  int64_t blk_stride, slot_stride, head_stride;
  int batch, groups, q_len, H, KVH, G;
  int bs, num_blocks, W, max_ctx;
  // page size, query rows a KV head and batch row, query heads a KV head, query heads, query
  // tokens, shares
  FastDiv by_bs, by_rps, by_g, by_h, by_q, by_shares;
  float scale_log2;
  // Workspace: the plan (for the merge) and the pieces' partials. A
  // unit's first piece goes to slot kind * rows + output row (kind 0: the group's segment, 1: the
  // row's own), a later one to slot 2 * rows + share * kShRows + row of the unit.
  int* plan;   // [sh_plan_words]
  float* ml;   // [slots][2]
  float* acc;  // [slots][D]
  int64_t rows;  // batch * q_len * H
  int shares;
};

// The plan's words: the cost of a share, then for each batch row, for the merge, what its own
// segment and its group's begin at and their 32-key blocks (none: 0), the group's first row and rows.
constexpr int kShPlanRows = 16, kShPlanRow = 8;
struct ShPlanRow {
  int own_cost, own_blocks, cost, blocks, first, members, pad[2];
};
static_assert(sizeof(ShPlanRow) == kShPlanRow * sizeof(int), "the plan's row");
__host__ __device__ constexpr int sh_plan_words(int batch) { return kShPlanRows + kShPlanRow * batch; }
__host__ __device__ constexpr int64_t sh_slots(int64_t rows, int shares) {
  return 2 * rows + static_cast<int64_t>(shares) * kShRows;
}

// As lds_copy16, with a cache policy.
template <int AUX>
__device__ __forceinline__ void sh_copy16(__amdgpu_buffer_rsrc_t r, char* dst, uint32_t voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 16, voff, 0, 0, AUX);
#endif
}
// A barrier of the workgroup that waits for LDS accesses only: the copies into LDS that are in
// flight stay so (__syncthreads would wait for them). What a wave copied is awaited by its own
// vmcnt before the barrier that publishes it.
__device__ __forceinline__ void sh_barrier() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#endif
}
// s_waitcnt immediate (gfx9 encoding): at most N vector memory operations outstanding.
constexpr int sh_wait_vm(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }

// `x`, from here on: what is found from it is not found ahead of the loops around, where it would hold
// registers that they need (22 in all; 16-bit caches at 128 dims spilled up to 19 without).
__device__ __forceinline__ int sh_here(int x) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(x));
#endif
  return x;
}

__device__ __forceinline__ void sh_here4(uint4& x) {
  x = make_uint4(sh_here(x.x), sh_here(x.y), sh_here(x.z), sh_here(x.w));
}
__device__ __forceinline__ void sh_here4(uint2& x) { x = make_uint2(sh_here(x.x), sh_here(x.y)); }

// The lane, found where it is asked for.
__device__ __forceinline__ int sh_lane() {
  return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, sh_here(0)));
}

// The least lo and the largest hi of each 16 lanes, one step: with those N lanes around.
template <int N>
__device__ __forceinline__ void sh_fold16(int& lo, int& hi) {
  lo = min(lo, __builtin_amdgcn_update_dpp(lo, lo, 0x120 + N, 0xF, 0xF, false));  // row_ror
  hi = max(hi, __builtin_amdgcn_update_dpp(hi, hi, 0x120 + N, 0xF, 0xF, false));
}

// 16-byte chunk c of a row of ROW bytes sits at chunk c ^ sh_swz(row): the 16 rows of a K operand
// read, and the rows of a transposed V read, then fall on distinct banks (pf_swz's patterns for
// rows of 256 and 128 bytes; rows of 64 bytes, four to a turn of the banks).
template <int ROW>
__device__ __forceinline__ int sh_swz(int r) {
  if constexpr (ROW >= 128) return pf_swz<ROW / 2>(r);
  return (r >> 2) & 3;
}

// Infinite values and NaN among the elements of a word of a cache row: the sign's place of each that
// is one. An exponent of ones (e4m3: all ones past the sign) carries into it.
template <typename KT>
__device__ __forceinline__ uint32_t sh_odd(uint32_t w) {
  constexpr uint32_t kOnes = sizeof(KT) == 1                   ? 0x7f7f7f7fu
                             : std::is_same<KT, bf16_t>::value ? 0x7f807f80u
                                                               : 0x7c007c00u;
  constexpr uint32_t kStep = sizeof(KT) == 1                   ? 0x01010101u
                             : std::is_same<KT, bf16_t>::value ? 0x00800080u
                                                               : 0x04000400u;
  return ((w & kOnes) + kStep) & (sizeof(KT) == 1 ? 0x80808080u : 0x80008000u);
}
template <typename T, typename KT>
__device__ __forceinline__ uint32_t sh_not_finite(const typename Kv8<T, KT>::raw_t& x) {
  uint32_t any = sh_odd<KT>(x.x) | sh_odd<KT>(x.y);
  if constexpr (sizeof(KT) != 1) any |= sh_odd<KT>(x.z) | sh_odd<KT>(x.w);
  return any;
}
// Zeros in their places.
template <typename T, typename KT>
__device__ __forceinline__ void sh_finite(typename Kv8<T, KT>::raw_t& x) {
  const auto clear = [](uint32_t& w) {
    const uint32_t odd = sh_odd<KT>(w);
    w &= ~(odd | (odd - (odd >> (8 * sizeof(KT) - 1))));
  };
  clear(x.x);
  clear(x.y);
  if constexpr (sizeof(KT) != 1) {
    clear(x.z);
    clear(x.w);
  }
}
// The mask of two 16-bit elements of which the first `n` are kept.
__device__ __forceinline__ uint32_t sh_pair_mask(int n) {
  return n >= 2 ? 0xffffffffu : (n == 1 ? 0xffffu : 0u);
}
// Ones of type T in the places of NaN and of the infinite values whose sign is `sign`'s, zeros
// elsewhere.
template <typename T>
__device__ __forceinline__ uint4 sh_ones(const uint4& x, uint32_t sign) {
  const auto ones = [sign](uint32_t w) {
    constexpr bool kB = std::is_same<T, bf16_t>::value;
    constexpr uint32_t kFraction = kB ? 0x007f007fu : 0x03ff03ffu;
    const uint32_t nan = ((w & kFraction) + kFraction) << (kB ? 8 : 5);  // (to the sign's place)
    return ((sh_odd<T>(w) & (nan | ~(w ^ sign))) >> 15) * (kB ? 0x3f80u : 0x3c00u);
  };
  return make_uint4(ones(x.x), ones(x.y), ones(x.z), ones(x.w));
}

template <typename T, typename KT, int D>
__global__ __launch_bounds__(kShThreads, 3) void shared_attn_kernel(const SharedParams p) {
  typedef Kv8<T, KT> KV;
  typedef ShCost<D, static_cast<int>(sizeof(KT))> Cost;
  static_assert(D == 64 || D == 128, "head_dim 64 and 128");
  constexpr int EB = static_cast<int>(sizeof(KT));
  constexpr bool FP8 = EB == 1;  // its rows are widened as the matrix operands are read
  constexpr int ROW = D * EB;             // bytes of a cache row
  constexpr int TK = sh_tile(D, EB);      // keys of a tile
  constexpr int SUB = TK / 16 / kShCopy;  // 16-key sub-tiles a copying wave brings
  constexpr int CPR = ROW / 16;           // 16-byte chunks a row
  constexpr int RPI = kWave / CPR;        // rows a copy instruction (1 KiB)
  constexpr int NI = 16 / RPI;            // copy instructions a sub-tile, of K and of V each
  constexpr int JD = D / 32;              // MFMA k-steps of a score block
  constexpr int ND = D / 16;              // 16-dim tiles of O^T
  static_assert(2 * SUB * NI == 16, "copy instructions a wave and tile");

  __shared__ __attribute__((aligned(256))) char s_tile[kShSlots * 2 * kShHalf];
  __shared__ int s_cum[2 * kShMaxBatch + 1];  // tiles before each segment: groups, then rows
  __shared__ int s_g0[kShMaxBatch + 1];       // a group's first row
  __shared__ int s_hi[kShMaxBatch];           // a group's prefix keys, 0 if no row reads them
  __shared__ int s_by[kShMaxBatch];           // the first row that does, whose table gives the pages
  __shared__ int s_len[kShMaxBatch];
  __shared__ int s_own[kShMaxBatch];          // where a row's own keys begin
  __shared__ short s_grp[kShMaxBatch];        // a row's group, or -1
  __shared__ float s_m[kShRows], s_l[kShRows];  // a piece's end: (m, l) of the computing waves' rows
  __shared__ int s_orow[kShRows];
  __shared__ __attribute__((aligned(8))) unsigned char s_live[kShSlots][kShCopy];  // sub-tiles in the slots that are no holes
  __shared__ int s_wsum[2 * (kShThreads / kWave)];
  __shared__ int s_edge[4];

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int g = lane >> 4;
  const int n = lane & 15;
  const int B = p.batch, NG = p.groups, NS = NG + B;
  const int RPS = p.q_len * p.G;  // query rows a KV head and batch row
  const auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };

  // ---- the plan: tiles and costs before each segment ----
  int* const s_cost = reinterpret_cast<int*>(s_tile);  // (until the first tile is brought)
  // (the first round's loads all at once: each is a miss to memory)
  int r0 = p.group_rows[min(tid, NG)], r1 = p.group_rows[min(tid + 1, NG)];
  int pages = p.prefix_pages[min(tid, NG - 1)], len = p.lens[min(tid, B - 1)];
  const auto row_in = [&](int r) { return r < 0 ? 0 : (r > B ? B : r); };
  bool descend = false;  // groups out of order: every row by itself
#pragma unroll 1
  for (int i = tid;;) {
    if (i <= NG) s_g0[i] = row_in(r0);
    if (i < NG) {
      const int64_t pt = static_cast<int64_t>(pages < 0 ? 0 : (pages > p.W ? p.W : pages)) * p.bs;
      s_cum[i] = static_cast<int>(pt < p.max_ctx ? pt : p.max_ctx);  // (for now: prefix tokens)
      s_hi[i] = 0;
      s_by[i] = B - 1;
      descend |= row_in(r0) > row_in(r1);
    }
    if (i < B) s_len[i] = len < 0 ? 0 : (len > p.max_ctx ? p.max_ctx : len);
    i += kShThreads;
    if (i > NG && i >= B) break;
    r0 = p.group_rows[min(i, NG)];
    r1 = p.group_rows[min(i + 1, NG)];
    pages = p.prefix_pages[min(i, NG - 1)];
    len = p.lens[min(i, B - 1)];
  }
  descend = __any(descend);
  if (lane == 0) s_wsum[w] = descend;
  __syncthreads();
  descend = __any(lane < kShThreads / kWave && s_wsum[lane] != 0);
#pragma unroll 1
  for (int b = tid; b < B; b += kShThreads) {
    int lo = 0, hi = NG;  // the last group that begins at or before row b
#pragma unroll 1
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_g0[mid] <= b) lo = mid; else hi = mid;
    }
    int own = 0, grp = -1;
    // (A group of one row has nothing to share: its prefix is the row's own. So is that of a row
    // whose queries do not all see it whole: what the others read past it, NaN perhaps, would
    // enter this row's sums with a weight of zero.)
    const int g0 = s_g0[lo], g1 = s_g0[lo + 1];
    if (!descend && g0 <= b && b < g1 && g1 - g0 > 1 && s_len[b] - p.q_len >= s_cum[lo] - 1) {
      own = s_cum[lo];
      grp = lo;
      s_hi[lo] = own;  // (every member's is the same)
      atomicMin(&s_by[lo], b);
    }
    s_own[b] = own;
    s_grp[b] = static_cast<short>(grp);
  }
  struct Segment {
    int b0, members, key0, hi, by;  // its first row and rows, its keys, the row whose table has them
  };
  auto segment = [&](int e) __attribute__((always_inline)) {
    const bool own = e >= NG;
    Segment x;
    x.b0 = own ? e - NG : s_g0[e];
    x.members = own ? 1 : s_g0[e + 1] - x.b0;
    x.key0 = own ? s_own[x.b0] : 0;
    x.hi = own ? s_len[x.b0] : s_hi[e];
    x.by = own ? x.b0 : s_by[e];
    return x;
  };
  int total = 0, total_cost = 0;  // the exclusive sums, a segment a thread
#pragma unroll 1
  for (int e0 = 0; e0 < NS; e0 += kShThreads) {
    __syncthreads();
    const int e = e0 + tid;
    int c = 0, cost = 0;
    if (e < NS) {  // (idle waves skip it)
      const Segment x = segment(e);
      const int blocks = (x.hi - x.key0 + 31) >> 5;
      if (blocks > 0) {
        const int units = p.KVH * ceil_div(x.members * RPS, kShRows);
        c = units * ceil_div(blocks, TK / 32);
        cost = units * (Cost::kPiece + blocks * Cost::block(x.members * RPS));
      }
    }
    const int incl = wave_inclusive_sum(c), incl_cost = wave_inclusive_sum(cost);
    if (lane == kWave - 1) {
      s_wsum[w] = incl;
      s_wsum[kShThreads / kWave + w] = incl_cost;
    }
    __syncthreads();
    // the waves' sums, scanned by lanes: tiles in lanes 0 .., costs from lane 32 on
    constexpr int NW = kShThreads / kWave;
    const int of = lane & 31;
    const int part = of < NW ? s_wsum[of + (lane >= 32 ? NW : 0)] : 0;
    const int scan = wave_inclusive_sum(part);
    const int tiles_before = w > 0 ? __builtin_amdgcn_readlane(scan, w - 1) : 0;
    const int all_tiles = __builtin_amdgcn_readlane(scan, 31);  // (lanes from 32 on count on top)
    const int cost_before = w > 0 ? __builtin_amdgcn_readlane(scan, 31 + w) - all_tiles : 0;
    const int at = total + tiles_before + incl - c, at_cost = total_cost + cost_before + incl_cost - cost;
    total += all_tiles;
    total_cost += __builtin_amdgcn_readlane(scan, 63) - all_tiles;
    if (e < NS) {
      s_cum[e] = at;
      s_cost[e] = at_cost;
    }
  }
  if (tid == 0) {
    s_cum[NS] = total;
    s_cost[NS] = total_cost;
  }
  __syncthreads();
  const int per = max(1, fast_quot(uni(total_cost) + p.shares - 1, p.by_shares));
  if (blockIdx.x == 0 && tid == 0) p.plan[0] = per;
#pragma unroll 1
  for (int b = static_cast<int>(blockIdx.x) + tid * p.shares; b < B; b += kShThreads * p.shares) {
    const int grp = s_grp[b];
    const Segment e = segment(grp < 0 ? 0 : grp);
    ShPlanRow* const o = reinterpret_cast<ShPlanRow*>(p.plan + kShPlanRows) + b;
    *reinterpret_cast<int4*>(o) =
        make_int4(s_cost[NG + b], max(0, (s_len[b] - s_own[b] + 31) >> 5), grp < 0 ? 0 : s_cost[grp],
                  grp < 0 ? 0 : (e.hi + 31) >> 5);
    *reinterpret_cast<int2*>(&o->first) = make_int2(e.b0, e.members);
  }
  // Contiguous shares to one XCD (workgroup i runs on XCD i % 8): the row blocks of one KV head
  // then read their keys through one L2.
  const int share = p.shares % kXcds == 0
                        ? static_cast<int>(blockIdx.x % kXcds) * (p.shares / kXcds) +
                              static_cast<int>(blockIdx.x / kXcds)
                        : static_cast<int>(blockIdx.x);
  // The share's tiles are those that begin at costs [share per, (share + 1) per): lane 0 of a wave
  // finds the first and its segment, lane 1 the next share's.
  if (w == 0) {
    int bound = total, lo = NS - 1;
    const int64_t edge = static_cast<int64_t>(share + (lane & 1)) * per;
    if (edge < total_cost) {
      const int x = static_cast<int>(edge);
      int hi = NS;  // the last segment that begins at or before x
      lo = 0;
#pragma unroll 1
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cost[mid] <= x) lo = mid; else hi = mid;
      }
      const Segment e = segment(lo);
      const uint32_t blocks = static_cast<uint32_t>((e.hi - e.key0 + 31) >> 5);
      const uint32_t step = static_cast<uint32_t>(Cost::block(e.members * RPS));
      const uint32_t unit_cost = Cost::kPiece + blocks * step;
      const uint32_t off = static_cast<uint32_t>(x - s_cost[lo]);
      const uint32_t unit = off / unit_cost;
      const int r = static_cast<int>(off - unit * unit_cost);
      const int tiles = ceil_div(static_cast<int>(blocks), TK / 32);
      const int t = r == 0 ? 0 : max(1, ceil_div(r - Cost::kPiece, static_cast<int>(step) * (TK / 32)));
      bound = s_cum[lo] + static_cast<int>(unit) * tiles + min(t, tiles);
    }
    if (lane < 2) {
      s_edge[lane] = bound;
      s_edge[2 + lane] = lo;
    }
  }
  __syncthreads();
  const int first = uni(s_edge[0]), last = uni(s_edge[1]);
  const int seg0 = uni(s_edge[2]), seg1 = uni(s_edge[3]) + 1;  // its segments
  if (first >= last) return;

  const bool copies = w >= kShComp;         // a copying wave
  const int cw = copies ? w - kShComp : w;  // its place among its side's

  // ---- a window of 64 tiles: lane i describes tile base + i ----
  // Everything the loops need of the plan is found here, each lane one tile, and later taken with
  // lane reads.
  //   tok  the key the tile begins at      hi  where the segment's keys end
  //   unit KV head | row block << 16       id  the pages of a copying wave's sub-tiles
  //   bits segment's first row | kind << 10 | the unit's first tile << 11 |
  //        the piece's last tile << 12 | (query rows - 1) << 13 | the piece's first tile << 20 |
  //        its keys are read for one row block only << 21 | the row whose table has them << 22
  struct Tile {
    int tok, hi, unit, bits;
    __device__ bool starts() const { return (bits >> 20) & 1; }
    __device__ bool ends() const { return (bits >> 12) & 1; }
    __device__ int rows() const { return ((bits >> 13) & 127) + 1; }
    // log2 of the computing waves that take different rows; the others take other keys of the same.
    __device__ int row_waves() const {
      return rows() > 64 ? 3 : (rows() > 32 ? 2 : (rows() > 16 ? 1 : 0));
    }
    // Pieces whose waves split the keys are joined through the slot.
    __device__ bool joins() const { return ends() && rows() <= 64; }
    __device__ int first_row() const { return bits & 1023; }
    __device__ int table_row() const { return static_cast<int>(static_cast<uint32_t>(bits) >> 22); }
    __device__ int kvh() const { return unit & 0xffff; }
    __device__ Tile at(int lane) const {
      return Tile{__builtin_amdgcn_readlane(tok, lane), __builtin_amdgcn_readlane(hi, lane),
                  __builtin_amdgcn_readlane(unit, lane), __builtin_amdgcn_readlane(bits, lane)};
    }
  };
  auto window = [&](int base) __attribute__((always_inline)) {
    const int pos = min(base + sh_lane(), last - 1);
    int lo = seg0, hi = seg1;  // the last segment that begins at or before pos
#pragma unroll 1
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cum[mid] <= pos) lo = mid; else hi = mid;
    }
    const bool own = lo >= NG;
    const Segment e = segment(lo);
    Tile c;
    c.hi = e.hi;
    const uint32_t tiles = static_cast<uint32_t>(ceil_div(e.hi - e.key0, TK));
    const uint32_t off = static_cast<uint32_t>(pos - s_cum[lo]);
    const uint32_t unit = off / tiles;
    const uint32_t t = off - unit * tiles;
    const uint32_t rtiles = static_cast<uint32_t>(ceil_div(e.members * RPS, kShRows));
    const uint32_t kvh = rtiles == 1 ? unit : unit / rtiles;
    const uint32_t rt = unit - kvh * rtiles;
    c.tok = e.key0 + static_cast<int>(t) * TK;
    c.unit = static_cast<int>(kvh | (rt << 16));
    c.bits = e.b0 | (own ? 1 << 10 : 0) | (t == 0 ? 1 << 11 : 0) |
             (t + 1 == tiles || pos + 1 == last ? 1 << 12 : 0) |
             ((min(kShRows, e.members * RPS - static_cast<int>(rt) * kShRows) - 1) << 13) |
             (t == 0 || pos == first ? 1 << 20 : 0) | (rtiles == 1 ? 1 << 21 : 0) |
             static_cast<int>(static_cast<uint32_t>(e.by) << 22);
    return c;
  };

  // Both sides meet, for each tile, at a barrier where it has landed and at one where its slot
  // has been read; at a piece's end, whose rows leave through the slot, at two more.
  int slot = 0;  // the tile's slot
  if (copies) {
    __builtin_amdgcn_s_setprio(2);
    // ================= the copying waves: SUB sub-tiles of K and of V each =================
#pragma unroll 1
    for (int wbase = first; wbase < last; wbase += kWave) {
      const int count = min(kWave, last - wbase);
      const Tile wt = window(wbase);
      int w_id[SUB];
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        const int tok = wt.tok + 16 * (SUB * cw + i);
        const int pg = fast_quot(tok, p.by_bs);
        w_id[i] = -1;
        if (tok < wt.hi && pg < p.W)
          w_id[i] = p.table[static_cast<int64_t>(wt.table_row()) * p.W + pg];
      }
      const int64_t row_bytes = p.slot_stride * EB;
      uint32_t dvo[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int lr = RPI * j + lane / CPR;
        dvo[j] = static_cast<uint32_t>(lr * row_bytes + 16 * ((lane % CPR) ^ sh_swz<ROW>(lr)));
      }
      int to = slot;  // the slot the next tile is brought to
      __builtin_amdgcn_s_waitcnt(sh_wait_vm(0));  // (the page ids: no later use waits for them)
#pragma unroll 1
      for (int i = -kShSlots; i < count; ++i) {
        if (i >= 0) {
          // tile i has landed: all but the copies of the tile after it
          __builtin_amdgcn_s_waitcnt(sh_wait_vm(16 * (kShSlots - 1)));
          sh_barrier();
          sh_barrier();  // it has been read
          if (wt.at(i).joins()) {
            sh_barrier();
            sh_barrier();
          }
          slot ^= 1;
        }
        const int r = i + kShSlots;  // the tile requested (past the window: nothing is read)
        const int rl = min(r, count - 1);
        const Tile c = wt.at(rl);
        const bool once = EB == 2 && ((c.bits >> 21) & 1);
        int live = 0;
        char* const d = s_tile + to * 2 * kShHalf + SUB * cw * 16 * ROW;
#pragma unroll
        for (int h = 0; h < SUB; ++h) {
          const int id = __builtin_amdgcn_readlane(w_id[h], rl);
          const bool in = r < count && id >= 0 && id < p.num_blocks;
          const int tok = c.tok + 16 * (SUB * cw + h);
          const int64_t o = static_cast<int64_t>(in ? id : 0) * p.blk_stride +
                            static_cast<int64_t>(tok - fast_quot(tok, p.by_bs) * p.bs) * p.slot_stride +
                            static_cast<int64_t>(c.kvh()) * p.head_stride;
          const int64_t off = static_cast<int64_t>(
              (static_cast<uint64_t>(static_cast<uint32_t>(uni(static_cast<int>(o >> 32)))) << 32) |
              static_cast<uint32_t>(uni(static_cast<int>(o))));
          const int nbytes = uni(in ? static_cast<int>((min(16, c.hi - tok) - 1) * row_bytes + ROW) : 0);
          const __amdgpu_buffer_rsrc_t rk = tile_rsrc(static_cast<const KT*>(p.k) + off, nbytes);
          const __amdgpu_buffer_rsrc_t rv = tile_rsrc(static_cast<const KT*>(p.v) + off, nbytes);
#pragma unroll
          for (int j = 0; j < NI; ++j) {
            if (once) {
              sh_copy16<kShAux>(rk, d + (16 * h + RPI * j) * ROW, dvo[j]);
              sh_copy16<kShAux>(rv, d + kShHalf + (16 * h + RPI * j) * ROW, dvo[j]);
            } else {
              sh_copy16<0>(rk, d + (16 * h + RPI * j) * ROW, dvo[j]);
              sh_copy16<0>(rv, d + kShHalf + (16 * h + RPI * j) * ROW, dvo[j]);
            }
          }
          if (in) live |= 1 << h;
        }
        if (lane == 0) s_live[to][cw] = static_cast<unsigned char>(live);
        to ^= 1;
      }
      // (the copies past the window read nothing, and have landed before its slots are used again)
      __builtin_amdgcn_s_waitcnt(sh_wait_vm(0));
    }
    return;
  }

  // ================= the computing waves =================
  uint4 qb[JD];  // B operands Q^T: row n, dims KV::qk_dim0(j, g) ..
  int orow = -1, hi_n = 0;  // its place in the output; it sees keys below hi_n
  int wave_all = 0, wave_any = 0;  // all rows of the wave see keys below wave_all, none past wave_any
  int RW = 1, rw = 0, ks = 0, KS = 1;  // the wave takes rows 16 rw .., every KS-th 32-key block
  bool unit_first = false;  // the piece holds its unit's first tile
  float m_run = -INFINITY, l_run = 0.0f;
  mf_f32x4 acc[ND];
#pragma unroll 1
  for (int wbase = first; wbase < last; wbase += kWave) {
    const int count = min(kWave, last - wbase);
    const Tile wt = window(wbase);
    // A negative scale goes into the query's sign, so that the largest score weighs most. (A scale
    // of zero weighs every visible key alike; a tiny one does the same and keeps the masked scores
    // infinite.)
    const float scale = fmaxf(fabsf(p.scale_log2), 1e-30f);
    const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
    const int vtok = FP8 ? 16 * (n >> 3) + 4 * g + ((n >> 1) & 3)  // the token a lane names in a
                         : 4 * g + (n >> 2);                       // transposed V read
#pragma unroll 1
    for (int i = -1; i < count; ++i) {  // (i == -1: before the window's first tile)
      const Tile c = wt.at(i < 0 ? 0 : i);
      char* const base = s_tile + slot * 2 * kShHalf;
      if (i >= 0) {
        sh_barrier();  // the tile has landed
        const uint32_t live4 = static_cast<uint32_t>(uni(*reinterpret_cast<const int*>(s_live[slot])));
        // (blocks past every row's last key, and a wave without rows, have nothing to do)
        const int blocks = min(TK / 32, (wave_any - c.tok + 31) >> 5);
#pragma unroll 1
        for (int kb = ks < KS ? ks : blocks; kb < blocks; kb += KS) {
          const int key = c.tok + 32 * kb;
          const int live = (live4 >> (8 * (2 * kb / SUB) + 2 * kb % SUB)) & 3;
          char* const kv = base + kb * 32 * ROW;
          mf_f32x4 s[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint4 kk[JD];
            const char* const row = kv + (16 * k + n) * ROW;
            if constexpr (FP8) {
#pragma unroll
              for (int j = 0; j < JD / 2; ++j) {
                const uint4 x = *reinterpret_cast<const uint4*>(row + 16 * ((4 * j + g) ^ sh_swz<ROW>(n)));
                kk[2 * j] = KV::operand(typename KV::raw_t{x.x, x.y});
                kk[2 * j + 1] = KV::operand(typename KV::raw_t{x.z, x.w});
              }
            } else {
#pragma unroll
              for (int j = 0; j < JD; ++j)
                kk[j] = *reinterpret_cast<const uint4*>(row + 16 * ((4 * j + g) ^ sh_swz<ROW>(n)));
            }
            s[k] = mf_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < JD; ++j) s[k] = Mfma16<T>::mac(kk[j], qb[j], s[k]);
          }
          // V^T, on its way during the softmax: tokens 4 g .. + 3 of the block's first 16 keys and of
          // its second, as pb holds them.
          typename KV::raw_t vv[ND];
#pragma unroll
          for (int u = 0; u < ND; ++u) {
            if constexpr (FP8) {
              char* const v = kv + kShHalf + vtok * ROW + 16 * (u ^ sh_swz<ROW>(vtok)) + 8 * (n & 1);
              typedef int sh_i2 __attribute__((ext_vector_type(2)));
              typedef __attribute__((address_space(3))) sh_i2 lds_i2;
              const sh_i2 a = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)v);
              vv[u] = typename KV::raw_t{static_cast<uint32_t>(a.x), static_cast<uint32_t>(a.y)};
            } else {
              char* const v = kv + kShHalf + vtok * ROW +
                              16 * ((2 * u + ((n & 3) >> 1)) ^ sh_swz<ROW>(vtok)) + 8 * (n & 1);
              const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)v));
              const uint2 b = __builtin_bit_cast(
                  uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(v + 16 * ROW)));
              vv[u] = typename KV::raw_t{a.x, a.y, b.x, b.y};
            }
          }
          __builtin_amdgcn_sched_barrier(0);
          if (key + 32 > wave_all || live != 3) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const bool ok = ((live >> k) & 1) && key + 16 * k + 4 * g + r < hi_n;
                s[k][r] = ok ? s[k][r] : -INFINITY;
              }
            // A key that other rows of the unit see and some of these do not (drafts): a weight of
            // zero times an infinite value or NaN would be NaN. Where the block holds one, the rows
            // that see it get it here, and the products take zero in its place. (Within 1.1 % of the
            // time without in 36 of 40 calls, 2.7 % at most, with what the registers cost; a branch
            // between softmax and products instead, a pass for each set of rows that see the same
            // keys, took up to 8 % over fp8.)
            if (wave_all < c.hi) {
              uint32_t odd = 0;
#pragma unroll
              for (int u = 0; u < ND; ++u) odd |= sh_not_finite<T, KT>(vv[u]);
              if (__builtin_expect(__any(odd != 0), 0)) {
                const int sees = hi_n - key - 4 * g;
                const uint32_t one2 = Pack2<T>::pack(1.0f, 1.0f);
                const uint4 seen = make_uint4(one2 & sh_pair_mask(sees), one2 & sh_pair_mask(sees - 2),
                                              one2 & sh_pair_mask(sees - 16), one2 & sh_pair_mask(sees - 18));
#pragma unroll
                for (int u = 0; u < ND; ++u) {
                  sh_here4(vv[u]);  // (what the test above found is not held for this)
#pragma unroll
                  for (int down = 0; down < 2; ++down) {
                    const mf_f32x4 has = Mfma16<T>::mac(sh_ones<T>(KV::operand(vv[u]), down ? 0x80008000u : 0u),
                                                        seen, mf_f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                      acc[u][r] += has[r] > 0.0f ? (down ? -INFINITY : INFINITY) : 0.0f;
                    __builtin_amdgcn_sched_barrier(0);
                  }
                  sh_finite<T, KT>(vv[u]);
                }
              }
            }
          }
          float mt = fmaxf(s[0][0], s[1][0]);
#pragma unroll
          for (int r = 1; r < 4; ++r) mt = fmaxf(mt, fmaxf(s[0][r], s[1][r]));
          mt = rows4_max(mt);
          // The running maximum moves, and what was summed is rescaled, only where a row's grew by
          // more than 8: weights reach 2^8 at most, and 32 products a block are mostly saved.
          mt *= scale;
          if (__any(mt > m_run + 8.0f)) {
            const float m_new = fmaxf(m_run, mt);
            const float alpha = m_run != -INFINITY ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int u = 0; u < ND; ++u) acc[u] *= alpha;
          }
          const float m_use = m_run != -INFINITY ? m_run : 0.0f;
          float pr[8];  // (masked scores weigh 2^-inf = 0, NaN stays NaN)
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              pr[4 * k + r] = __builtin_amdgcn_exp2f(fmaf(s[k][r], scale, -m_use));
          // The weights are rounded to the query type for the matrix cores (half a step of it); l
          // sums the rounded ones, so that the weights used still sum to one.
          const uint4 pb = make_uint4(Pack2<T>::pack(pr[0], pr[1]), Pack2<T>::pack(pr[2], pr[3]),
                                      Pack2<T>::pack(pr[4], pr[5]), Pack2<T>::pack(pr[6], pr[7]));
          const uint32_t one2 = Pack2<T>::pack(1.0f, 1.0f);
          l_run += Dot2<T>::dot(pb.w, one2, Dot2<T>::dot(pb.z, one2, 0.0f)) +
                   Dot2<T>::dot(pb.y, one2, Dot2<T>::dot(pb.x, one2, 0.0f));
#pragma unroll
          for (int u = 0; u < ND; ++u) acc[u] = Mfma16<T>::mac(KV::operand(vv[u]), pb, acc[u]);
        }
      }

      // ---- the next piece's query rows are requested here (its first tile is the next one), ahead
      // of the copies that follow the barrier ----
      const bool ends = i >= 0 && c.ends();
      const bool next = i + 1 < count;
      const Tile nx = wt.at(next ? i + 1 : 0);
      const bool starts = next && nx.starts();
      int n_row = -1, n_hi = 0;  // the row requested
      uint4 nq[JD];
      if (starts) {
        const int b0 = nx.first_row();
        const T* const q = static_cast<const T*>(p.q) + static_cast<int64_t>(b0) * p.q_len * p.H * D;
        const int r = 16 * (cw & ((1 << nx.row_waves()) - 1)) + n;
        const int row = (nx.unit >> 16) * kShRows + (r < nx.rows() ? r : 0);
        const int member = fast_quot(row, p.by_rps);
        const int rest = row - member * RPS;
        const int tq = fast_quot(rest, p.by_g);
        const int o = (member * p.q_len + tq) * p.H + nx.kvh() * p.G + (rest - tq * p.G);
        const int at_g = sh_here(g);
#pragma unroll
        for (int j = 0; j < JD; ++j)
          nq[j] = *reinterpret_cast<const uint4*>(q + static_cast<int64_t>(o) * D +
                                                  KV::qk_dim0(j, at_g, JD));
        if (r < nx.rows()) {
          n_row = b0 * p.q_len * p.H + o;
          n_hi = min(nx.hi, s_len[b0 + member] - p.q_len + tq + 1);
        }
      }
      if (i >= 0) {
        sh_barrier();  // the slot has been read
        slot ^= 1;
      }
      // ---- a piece's end: its partials ----
      const int64_t slot0 = unit_first ? ((c.bits >> 10) & 1) * p.rows
                                       : 2 * p.rows + static_cast<int64_t>(share) * kShRows;
      const int rr = 16 * rw + n;  // the lane's row of the unit
      const float l = rows4_sum(l_run);
      const bool joins = ends && KS > 1;
      float* const f = reinterpret_cast<float*>(base);
      if (joins) {
        // Waves that split the keys put theirs into the slot: row rr of key wave ks at row
        // 16 RW ks + rr, its 16-byte chunk j at chunk j ^ n (the lanes of a set hold 16 rows).
        const int at = 16 * RW * ks + rr;
        const int chunk = sh_here(n);
        if (rr < c.rows() && ks < KS) {
#pragma unroll
          for (int u = 0; u < ND; ++u)
            *reinterpret_cast<float4*>(f + at * D + 4 * ((4 * u + g) ^ chunk)) =
                make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
          if (g == 0) {
            s_m[at] = m_run;
            s_l[at] = l;
            if (ks == 0) s_orow[rr] = orow;
          }
        }
        sh_barrier();
      }
      // (the query has arrived before the partials' stores, which a later wait would wait for too)
      __builtin_amdgcn_s_waitcnt(sh_wait_vm(0));
      if (starts) {
#pragma unroll
        for (int j = 0; j < JD; ++j) {
          qb[j] = make_uint4(nq[j].x ^ flip, nq[j].y ^ flip, nq[j].z ^ flip, nq[j].w ^ flip);
          keep_here(qb[j]);
        }
      }
      if (ends && !joins && orow >= 0) {
        const int64_t at = slot0 + (unit_first ? orow : rr);
        const int at_g = sh_here(g);
        if (g == 0) *reinterpret_cast<float2*>(p.ml + 2 * at) = make_float2(m_run, l);
#pragma unroll
        for (int u = 0; u < ND; ++u)
          *reinterpret_cast<float4*>(p.acc + at * D + 16 * u + 4 * at_g) =
              make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
      }
      if (joins) {  // a thread joins 4 dims of a row
#pragma unroll 1
        for (int x = kWave * cw + sh_lane(); x < c.rows() * (D / 4); x += kShComp * kWave) {
          const int r = x / (D / 4), j = x % (D / 4);
          float M = -INFINITY;
#pragma unroll
          for (int k = 0; k < kShComp; ++k) M = fmaxf(M, s_m[(k < KS ? k : 0) * 16 * RW + r]);
          const float m_use = M != -INFINITY ? M : 0.0f;
          float L = 0.0f;
          float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
          for (int k0 = 0; k0 < KS; k0 += 2) {  // (KS is 2, 4 or 8)
#pragma unroll
            for (int k = k0; k < k0 + 2; ++k) {
              const int at = k * 16 * RW + r;
              const float e = __builtin_amdgcn_exp2f(s_m[at] - m_use);
              const float4 y = *reinterpret_cast<const float4*>(f + at * D + 4 * (j ^ (r & 15)));
              L = fmaf(s_l[at], e, L);
              o.x = fmaf(y.x, e, o.x);
              o.y = fmaf(y.y, e, o.y);
              o.z = fmaf(y.z, e, o.z);
              o.w = fmaf(y.w, e, o.w);
            }
          }
          const int64_t at = slot0 + (unit_first ? s_orow[r] : r);
          if (j == 0) *reinterpret_cast<float2*>(p.ml + 2 * at) = make_float2(M, L);
          *reinterpret_cast<float4*>(p.acc + at * D + 4 * j) = o;
        }
        sh_barrier();  // the slot is free
      }
      // ---- the next piece begins ----
      if (starts) {
        unit_first = (nx.bits >> 11) & 1;
        RW = 1 << nx.row_waves();
        rw = cw & (RW - 1);
        KS = min(kShComp >> nx.row_waves(), TK / 32);  // (waves ks >= KS have no block)
        ks = cw >> nx.row_waves();
        orow = n_row;
        hi_n = n_hi;
        m_run = -INFINITY;
        l_run = 0.0f;
#pragma unroll
        for (int u = 0; u < ND; ++u) acc[u] = mf_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        int lo = orow < 0 ? INT_MAX : hi_n, hi = hi_n;
        sh_fold16<8>(lo, hi);
        sh_fold16<4>(lo, hi);
        sh_fold16<2>(lo, hi);
        sh_fold16<1>(lo, hi);
        wave_all = uni(lo);
        wave_any = uni(hi);
      }
    }
  }
}

// Joins a row's pieces: one wave a query row, D / 64 dims a lane. Its pieces: for the group's
// segment (if the row has one) and for its own, the unit's first piece, then those of the shares
// that the unit runs on into. A lane finds one piece each and its weight; the accumulators follow.
constexpr int kShMergeThreads = 256;
constexpr int kShMergeWaves = kShMergeThreads / kWave;
template <typename T, int D, int EB>
__global__ __launch_bounds__(kShMergeThreads) void shared_merge_kernel(const SharedParams p) {
  typedef ShCost<D, EB> Cost;
  constexpr int TB = sh_tile(D, EB) / 32;  // 32-key blocks of a tile
  constexpr int DPL = D / 64;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kShMergeWaves +
                      __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  if (row >= p.rows) return;
  const int per = p.plan[0];
  const int bi = fast_quot(static_cast<int>(row), p.by_h);
  const int b = fast_quot(bi, p.by_q), i = bi - b * p.q_len;
  const int h = static_cast<int>(row) - bi * p.H;
  const int kvh = fast_quot(h, p.by_g);
  const int r0 = i * p.G + h - kvh * p.G;
  const int RPS = p.q_len * p.G;
  const ShPlanRow e = reinterpret_cast<const ShPlanRow*>(p.plan + kShPlanRows)[b];
  // A unit's pieces: the first at the row's own place, the others at the places of the shares up to
  // the last tile's one (but for shares so small that they hold no tile of the unit).
  struct Unit {
    int begin, tile, last, r, share, pieces;  // its cost, a tile's, the last tile, the row in it,
  };                                          // the first tile's share, shares to the last's
  const auto share_of = [&](int cost) {
    return static_cast<int>(static_cast<uint32_t>(cost) / static_cast<uint32_t>(per));
  };
  const auto unit = [&](int cost, int blocks, int r, int members) __attribute__((always_inline)) {
    const int step = Cost::block(members * RPS);
    const int rtiles = (members * RPS + kShRows - 1) / kShRows;
    Unit u;
    u.begin = cost + (kvh * rtiles + r / kShRows) * (Cost::kPiece + blocks * step);
    u.tile = TB * step;
    u.last = (blocks - 1) / TB;
    u.r = r % kShRows;
    u.share = share_of(u.begin);
    u.pieces = blocks <= 0 ? 0
               : u.last == 0 ? 1
                             : share_of(u.begin + Cost::kPiece + u.last * u.tile) - u.share + 1;
    return u;
  };
  const Unit group = unit(e.cost, e.blocks, (b - e.first) * RPS + r0, e.members);
  const Unit own = unit(e.own_cost, e.own_blocks, r0, 1);
  float M = -INFINITY, L = 0.0f;
  float o[DPL];
#pragma unroll
  for (int d = 0; d < DPL; ++d) o[d] = 0.0f;
#pragma unroll 1
  for (int base = 0; base < group.pieces + own.pieces; base += kWave) {
    // a lane a piece: its place, its maximum and its weight
    const bool first = base + lane < group.pieces;
    const int k = base + lane - (first ? 0 : group.pieces);
    const int begin = first ? group.begin : own.begin, tile = first ? group.tile : own.tile;
    const int share = (first ? group.share : own.share) + k;
    const int past = share * per - begin - Cost::kPiece;  // the share's first tile
    const int t = past <= tile ? 1
                               : static_cast<int>(static_cast<uint32_t>(past + tile - 1) /
                                                  static_cast<uint32_t>(tile));
    const bool on = first || k < own.pieces;
    const bool holds = k == 0 || (t <= (first ? group.last : own.last) &&
                                  begin + Cost::kPiece + t * tile < (share + 1) * per);
    const int64_t place =
        !(on && holds) ? 0
        : k == 0       ? (first ? row : p.rows + row)
                       : 2 * p.rows + static_cast<int64_t>(share) * kShRows + (first ? group.r : own.r);
    const float2 ml = *reinterpret_cast<const float2*>(p.ml + 2 * place);
    uint64_t mask = __ballot(on && holds);
    float mx = on && holds ? ml.x : -INFINITY;
    mx = fmaxf(M, group_max<kWave>(mx));
    const bool some = mx != -INFINITY;
    const float w = !(on && holds) ? 0.0f : (some ? __builtin_amdgcn_exp2f(ml.x - mx) : 0.0f);
    const float w0 = some ? __builtin_amdgcn_exp2f(M - mx) : 1.0f;
    L = fmaf(L, w0, group_sum<kWave>(on && holds ? ml.y * w : 0.0f));
    M = mx;
#pragma unroll
    for (int d = 0; d < DPL; ++d) o[d] *= w0;
#pragma unroll 1
    while (mask != 0) {  // the pieces' accumulators, eight on their way at once
      constexpr int N = 8;
      float a[N][DPL], wk[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool have = mask != 0;
        const int l = have ? __builtin_ctzll(mask) : 0;
        mask &= mask - 1;
        const int64_t at = have ? static_cast<int64_t>(
            static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(place >> 32), l))) << 32 |
            static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(place), l))) : 0;
        wk[i] = have ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), l)) : 0.0f;
        const float* const src = p.acc + at * D + DPL * lane;
#pragma unroll
        for (int d = 0; d < DPL; ++d) a[i][d] = have ? src[d] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int d = 0; d < DPL; ++d) o[d] = fmaf(a[i][d], wk[i], o[d]);
    }
  }
  const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);
  T* const out = static_cast<T*>(p.out) + row * D + DPL * lane;
#pragma unroll
  for (int d = 0; d < DPL; ++d) Elt<T>::store(out + d, o[d] * inv);
}

template <typename T, typename KT>
hipError_t launch_shared(const SharedParams& p, int D, hipStream_t stream);

#define MSATTN_DECLARE_SHARED(T, KT) \
  template <>                        \
  hipError_t launch_shared<T, KT>(const SharedParams& p, int D, hipStream_t stream);
MSATTN_DECLARE_SHARED(bf16_t, bf16_t)
MSATTN_DECLARE_SHARED(_Float16, _Float16)
MSATTN_DECLARE_SHARED(bf16_t, fp8_t)
MSATTN_DECLARE_SHARED(_Float16, fp8_t)
#undef MSATTN_DECLARE_SHARED

template <typename T, typename KT, int D>
hipError_t launch_shared_one(const SharedParams& p, hipStream_t stream) {
  hipLaunchKernelGGL((shared_attn_kernel<T, KT, D>), dim3(static_cast<unsigned>(p.shares)),
                     dim3(kShThreads), 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t blocks = (p.rows + kShMergeWaves - 1) / kShMergeWaves;
  hipLaunchKernelGGL((shared_merge_kernel<T, D, sizeof(KT)>), dim3(static_cast<unsigned>(blocks)),
                     dim3(kShMergeThreads), 0, stream, p);
  return hipGetLastError();
}

#define MSATTN_DEFINE_SHARED(T, KT)                                                      \
  template <>                                                                            \
  hipError_t launch_shared<T, KT>(const SharedParams& p, int D, hipStream_t stream) {    \
    return D == 128 ? launch_shared_one<T, KT, 128>(p, stream)                           \
                    : launch_shared_one<T, KT, 64>(p, stream);                           \
  }

}  // namespace msattn
