// Attention over the 4-bit paged cache (fp4_cache.h; gfx950): any query type, any q_len.
//
// A unit is a (batch row, KV head, block of up to 16 CT query rows); rows are the pairs (query
// token i, head g of the KV head's group) r = i G + g. Its keys are cut into groups of 32 tokens
// (two tiles). A workgroup has 8 waves, two a SIMD, and units come to it in one of three ways
// (plan_of in abi_fp4.hip chooses, by what each costs):
//   list   all groups of all units, in order, a unit's behind kFp4Head empty positions, are cut
//          into one contiguous share a CU, whatever the lengths (read on the device, so a call is
//          capture-safe). A workgroup's waves take its share's groups in turn, and go on from unit
//          to unit without waiting for each other. For more units than CUs, long and ragged: 64 rows
//          of 1024 to 8192 keys of H32/KVH8/D128 take 50 us, 4.3 TB/s of the cache, 5.4 to 6.8 inside
//          a share.
//   parts  a unit is cut into equal parts, a workgroup each, joined as shares are but without a
//          plan. For few long units: 16 rows of 1024 to 4096 keys of H28/KVH4/D128 in fp16 take 16
//          us, as a list 20.7.
//   dealt  a unit is whole: WK waves take its groups in turn, and 8 / WK units share a workgroup.
//          For chunks of prompts, with thousands of units, and for short contexts: no plan, no
//          partials and no joins.
// What a wave or a share leaves of a unit is, for each query row,
//   m,  l = sum_j 2^(s_j - m),  acc = sum_j 2^(s_j - m) V_j,   s_j = scale log2(e) q.K_j
// over its visible keys. The waves' parts are joined in LDS; a unit that lies within one share is then
// normalised and written, the shares of another leave partials in the workspace, and the last of them
// to arrive joins them; so too with parts.
//
// A wave loads a tile's keys and values straight into the registers of the matrix operands, 16
// bytes a lane, contiguous (fp4_cache.h); the next kRing groups are on their way while it works on
// one. Lane (g, n) = (l / 16, l % 16):
//   * S^T = K Q^T on v_mfma_f32_16x16x32_bf16: the lane holds 32 dims of key n of the tile (at
//     D = 128), widened by v_cvt_scalef32_pk_bf16_fp4, which is exact, and the same dims of query
//     row n; it receives row n's scores of keys 4 g .. 4 g + 3 of the tile.
//   * Those of the group's two tiles, 8 weights, are in their lane the B operand of
//     O^T += V^T P^T; the A operand is the 8 dims the lane holds of the same 8 tokens, so that
//     product c takes dim 8 n + c and the lane receives dims 32 g .. 32 g + 31 of row n. Softmax and
//     rescaling stay in the lane.
// The scaled 4-bit matrix instructions are not used: with an e4m3 operand beside the 4-bit one,
// sums of 128 products came out up to 9e-5 of the sum of magnitudes off, bf16 ones exactly rounded.
//
// What bounds it. A decode: the cache's bytes in the middle of a share, and about 7 us of start (the
// plan, the table, the first tiles) and end (parts and joins) around it, all there is to a small call.
// A chunk: the widening. A tile is widened once for each unit that reads it, so units of few rows spend
// their time on it, 64 a wave (CT = 4, their query in LDS) less than 32 in registers (abi_fp4.hip has
// both sides).
//
// fp16 and fp32 queries enter the products as 2 and 3 bf16 parts, which hold all their digits; weights,
// which are fp32, as 2 parts for 16-bit queries and 3 for fp32 ones (16 and 24 digits). Maxima, sums and
// accumulators are fp32. (One part was rounded to 8 digits, whose error in a bf16 answer, a mean of
// values weighed so, was as large as the answer's own rounding: mean relative error against 64 bits
// 0.0023, with two parts 0.0017. 512 queries of H28/KVH4/D128 behind 4096 keys, two rows of them, take
// 103 us with two parts, 92 with one; decodes are level. The chunk in fp16 126 us, in fp32 194.)
//
// A masked key's score is -inf, and where a group has masked keys, values that some row must not see
// are taken as zeros, and their NaN, if any, is given to the rows that do see them.
//
// Semantics: miniserve/attention.py:205-250.
#pragma once

#include "decode_mfma.h"
#include "fp4_cache.h"

#define FP4_INLINE __attribute__((always_inline))

namespace msattn {

constexpr int kFp4Waves = 8;             // waves of a workgroup, two a SIMD
constexpr int kFp4Threads = 64 * kFp4Waves;
constexpr int kFp4Group = 32;            // tokens of a group
constexpr int kFp4MaxEntries = 2048;     // (row, row block) pairs whose shares are planned in LDS
constexpr int kFp4Shares = 256;          // of a list, at most: one a CU, an arrival counter each
static_assert(kFp4Shares <= kMaxTickets, "a counter a share");
// Positions of the list ahead of a unit's groups that hold no work: what its start and end cost a
// workgroup, in groups. Without them a share of many short units ends last: 64 rows of H32/KVH8/D128
// with 1024 to 8192 keys, 0, 8, 24 and 48 of them, 58.2, 52.8, 50.0 and 52.0 us; with 4096 each, where
// every share has the same, 56.6, 56.7, 57.7 and 57.2.
constexpr int kFp4Head = 24;

struct Fp4Params {
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  const int32_t* table;
  const int32_t* lens;
  void* out;
  int64_t blk_stride, head_stride;  // bytes
  int64_t q_st[3];                  // batch, token and head strides of the query (elements)
  int batch, q_len, H, KVH, G, D;
  int bs, num_blocks, W, max_ctx;
  int causal, window;
  float scale_log2;
  int rows_per_kvh;  // q_len * G
  int rblocks;       // ceil(rows_per_kvh / (16 CT))
  int slot_rows;     // rows of a partial: min(16 CT, rows_per_kvh)
  int xcd_units;     // without a list: workgroups an XCD
  int shares;        // of a list
  int parts;         // of a unit
  Fp4Div by_tiles;   // tiles of a page
  Fp4Div by_g, by_rb, by_kvh, by_parts;
  Fp4Div by_per;     // D / 4
  int* tickets;
  float* ml;         // [2 shares][slot_rows][2]
  float* acc;        // [2 shares][slot_rows][D]
};

// A value the compiler knows nothing of from here on.
__device__ __forceinline__ void opaque(uint32_t& x) {
#if defined(__HIP_DEVICE_COMPILE__)  // the constraint names a GPU register class
  asm volatile("" : "+v"(x));
#endif
}

// bf16 parts that a T's value enters a product as.
template <typename T> constexpr int fp4_parts() {
  return std::is_same<T, bf16_t>::value ? 1 : (std::is_same<T, _Float16>::value ? 2 : 3);
}

// One packed pair of bf16 parts of a and b, cut off (not rounded, so that no part overflows), and
// what is left of them. A part that is not finite leaves nothing. (A NaN is made quiet: one whose
// payload lies in the lower half alone would be cut to an infinity.)
__device__ __forceinline__ uint32_t fp4_cut2(float& a, float& b) {
  const uint32_t x = (__float_as_uint(a) | (a != a ? 0x400000u : 0u)) & 0xffff0000u;
  const uint32_t y = (__float_as_uint(b) | (b != b ? 0x400000u : 0u)) & 0xffff0000u;
  a = (x & 0x7f800000u) == 0x7f800000u ? 0.0f : a - __uint_as_float(x);
  b = (y & 0x7f800000u) == 0x7f800000u ? 0.0f : b - __uint_as_float(y);
  return (x >> 16) | y;
}

// The same of finite weights (or NaN), each part rounded to nearest: what is left has as many digits
// less, and a sign, and is exact (a dot product with (-1, 0) or (0, -1) takes a part away; the other
// weight of the pair is the same row's, so that its NaN changes no answer. 2 x 512 fp16 queries behind
// 4096 keys: cut off 162 us, rounded 147, with the dot products 126 against 139).
__device__ __forceinline__ uint32_t fp4_part2(float& a, float& b) {
  const uint32_t w = Pack2<bf16_t>::pack(a, b);
  uint32_t first = 0x0000bf80u;  // (-1, 0)
#if defined(__HIP_DEVICE_COMPILE__)
  asm("" : "+s"(first));  // (as a constant it is encoded as -1.0f, which is (0, -1))
#endif
  a = Dot2<bf16_t>::dot(w, first, a);
  b = Dot2<bf16_t>::dot(w, 0xbf800000u, b);
  return w;
}

// Byte S of w, two 4-bit elements, as two bf16 times scale.
template <int S>
__device__ __forceinline__ uint32_t fp4_widen2(uint32_t w, float scale) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const b2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, S);
  return __builtin_bit_cast(uint32_t, r);
}

// Four neighbouring outputs (on 4 elements' alignment), rounded to nearest.
template <typename T>
__device__ __forceinline__ void fp4_store4(T* o, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(o) = make_float4(a, b, c, d);
  else *reinterpret_cast<uint2*>(o) = make_uint2(Pack2<T>::pack(a, b), Pack2<T>::pack(c, d));
}

// A lane's bytes of a tile, through the tile's descriptor. (Nontemporal loads took 61 -> 73 us on 64
// rows of H32/KVH8/D128: a tile's first and last lines are its neighbours' too.)
template <typename V>
__device__ __forceinline__ V fp4_load(__amdgpu_buffer_rsrc_t r, uint32_t at) {
  const int off = static_cast<int>(at);
  if constexpr (sizeof(V) == 16) {
    const mf_u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
    return V{x.x, x.y, x.z, x.w};
  } else if constexpr (sizeof(V) == 8) {
    typedef uint32_t u2 __attribute__((ext_vector_type(2)));
    const u2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
    return V{x.x, x.y};
  } else if constexpr (sizeof(V) == 4) {
    return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  } else {
    return __builtin_amdgcn_raw_buffer_load_b8(r, off, 0, 0);
  }
}

// The power of two of byte i of w, as the widening instruction takes it: it reads the exponent's bits
// alone (checked on all bytes, whatever the others).
__device__ __forceinline__ float fp4_scale_of(uint32_t w, int i) {
  return __uint_as_float(i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1);
}

// Keys a query row, and a block of rows, may see, and a unit's place in the work list.
struct Fp4Unit {
  int b, kvh, rb;
  int ctx;           // the row's context
  int lo, hi;        // keys that some row of the block sees
  int first, n;      // its groups of keys
  int u0;            // position of its first group in the list
  // Of the share: the unit's groups skip .. skip + cnt - 1, which are the share's r0 .. r0 + cnt - 1
  int skip, cnt, r0;
};

template <int ROWS>
__device__ __forceinline__ void fp4_extent(const Fp4Params& p, int ctx, int rb, int* lo, int* hi) {
  const int r0 = rb * ROWS;
  const int r1 = min(r0 + ROWS, p.rows_per_kvh) - 1;
  const int q0 = ctx - p.q_len + fp4_quot(r0, p.by_g), q1 = ctx - p.q_len + fp4_quot(r1, p.by_g);
  *hi = p.causal ? max(0, min(ctx, q1 + 1)) : ctx;
  *lo = p.window > 0 ? max(0, q0 - p.window + 1) : 0;
  if (*lo > *hi) *lo = *hi;
}
__device__ __forceinline__ int fp4_first(int lo) { return lo / kFp4Group; }
__device__ __forceinline__ int fp4_count(int lo, int hi) {  // at least one, so that zeros are written
  return hi > lo ? ceil_div(hi, kFp4Group) - lo / kFp4Group : 1;
}

// How units come to the workgroups.
enum : int { kFp4Dealt, kFp4Parts, kFp4List };

// WK waves take a unit's groups in turn. WAY = kFp4List (WK = 8): a workgroup takes a share of the list;
// kFp4Parts (WK = 8): one of p.parts parts of a unit; else 8 / WK units, neighbours in the list.
template <typename T, int DP, int CT, int WK, int WAY>
__global__ __launch_bounds__(kFp4Threads, 2) void fp4_attn_kernel(const Fp4Params p) {
  constexpr bool LIST = WAY == kFp4List, PARTS = WAY == kFp4Parts;
  static_assert(WAY == kFp4Dealt || WK == kFp4Waves, "a share's groups are all waves'");
  constexpr int HV = DP > 128 ? 2 : 1;   // halves of 128 dims
  constexpr int DH = DP > 128 ? 128 : DP;
  constexpr int NJ = DH / 32;            // score products of a half; dwords of keys a lane holds
  constexpr int VC = DH / 16;            // value products of a half: dims a lane holds of a token
  constexpr int LD = DH / 4;             // dims a lane receives of a half
  constexpr int PQ = fp4_parts<T>();
  constexpr int PW = PQ == 1 ? 2 : PQ;   // bf16 parts of a weight
  constexpr int ROWS = 16 * CT;
  constexpr bool QLDS = CT == 4;         // the query's operands in LDS, where a unit's waves share them
  // Groups on their way while one is worked on: as many as the registers hold. With CT = 4 one, its
  // keys requested as soon as the group before has used its own, before that one's softmax.
  // Three where a list streams; two are enough for a unit or a part of one, which begins with all of them
  // (64 rows of H32/KVH8/D128 up to 1300 keys, two, three and four: 24.1, 25.8, 27.9 us).
  constexpr int kRing = QLDS || (DP == 256 && PQ > 1) ? 1
                        : !LIST || DP == 256 || (CT == 2 && PQ == 3) ? 2 : 3;
  constexpr bool kEarly = kRing == 1;
  typedef typename std::conditional<DH == 128, uint4, uint2>::type kraw_t;

  __shared__ int s_pre[LIST ? kFp4MaxEntries + 1 : 1];
  __shared__ int s_ctx[LIST ? kFp4MaxEntries : 1];
  __shared__ int s_tot[kFp4Waves];  // and whether this workgroup joins a unit's shares
  // The waves' accumulators of up to 16 rows of a unit, [buffer][wave][rows][RS] (RS: the rows of a
  // store fall on different banks), and their maxima and sums. Fewer rows leave more buffers.
  constexpr int RS = DP + 4;
  constexpr int kAccWords = kFp4Waves * 16 * RS, kQueryWords = QLDS ? kFp4Waves / WK * CT * HV * NJ * 64 * 4 : 0;
  __shared__ __attribute__((aligned(16))) float
      s_acc[kAccWords > kQueryWords ? kAccWords : kQueryWords];  // (and the query's operands before)
  __shared__ float2 s_ml[kFp4Waves * 16];
  __shared__ int s_prog[kFp4Waves];  // groups that a wave has taken
  __shared__ int s_first[5];         // the share's first unit
  __shared__ int s_cnt[16], s_done[16];  // of a buffer: waves that have written it, times it was read

  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, n = lane & 15;
  const int share = static_cast<int>(blockIdx.x);
  constexpr int NU = kFp4Waves / WK;        // units at a time
  const int wu = w / WK, wk = w % WK;       // the wave's unit, and its place among the unit's waves
  const int entries = p.batch * p.rblocks;

  // Barrier for what lies in LDS: loads into registers stay on their way.
  auto lds_barrier = [&]() FP4_INLINE {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  if (tid < 16) s_cnt[tid] = s_done[tid] = 0;
  if (tid < kFp4Waves) s_prog[tid] = 0;
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  auto clamped = [&](int c) FP4_INLINE { return c < 0 ? 0 : (c > p.max_ctx ? p.max_ctx : c); };
  // The list: groups of one head's units of entries 0 .. e - 1 (entry = row, row block). A batch of
  // up to 64 rows of one block each has it in registers, entry e's sum with its own groups and its
  // context in lane e of every wave; others in LDS.
  const bool regs = p.rblocks == 1 && p.batch <= 64;
  int c0 = 0, c1 = 0, chunk = 1, lane_sum = 0, lane_ctx = 0;
  if constexpr (LIST) {
    int sum = 0;
    if (regs) {
      int cnt = 0;
      if (lane < p.batch) {
        lane_ctx = clamped(p.lens[lane]);
        int lo, hi;
        fp4_extent<ROWS>(p, lane_ctx, 0, &lo, &hi);
        cnt = fp4_count(lo, hi) + kFp4Head;
      }
      lane_sum = wave_inclusive_sum(cnt);
      sum = __builtin_amdgcn_readlane(lane_sum, 63);
    } else {
      for (int e0 = 0; e0 < entries; e0 += kFp4Threads) {
        const int e = e0 + tid;
        int cnt = 0;
        if (e < entries) {
          const int b = fp4_quot(e, p.by_rb), rb = e - b * p.rblocks, ctx = clamped(p.lens[b]);
          if (rb == 0) s_ctx[b] = ctx;
          int lo, hi;
          fp4_extent<ROWS>(p, ctx, rb, &lo, &hi);
          cnt = fp4_count(lo, hi) + kFp4Head;
        }
        const int incl = wave_inclusive_sum(cnt);
        if (lane == 63) s_tot[w] = incl;
        __syncthreads();
        int before = sum;
#pragma unroll
        for (int i = 0; i < kFp4Waves; ++i) {
          const int t = s_tot[i];
          if (i < w) before += t;
          sum += t;
        }
        if (e < entries) s_pre[e + 1] = before + incl;
        if (e == 0) s_pre[0] = 0;
        __syncthreads();
      }
      sum = uniform(sum);
    }
    const int total = sum * p.KVH;
    // (whole rounds of the waves)
    chunk = ceil_div(ceil_div(total, p.shares), kFp4Waves) * kFp4Waves;
    c0 = static_cast<int>(min(static_cast<int64_t>(share) * chunk, static_cast<int64_t>(total)));
    c1 = min(c0 + chunk, total);
    if (c0 >= c1) return;  // (the workgroup as one)
  }
  auto sum_before = [&](int e) FP4_INLINE {
    if (!regs) return uniform(s_pre[e]);
    return e == 0 ? 0 : __builtin_amdgcn_readlane(lane_sum, e - 1);
  };
  auto context = [&](int b) FP4_INLINE {
    if constexpr (!LIST) return uniform(clamped(p.lens[b]));
    return regs ? __builtin_amdgcn_readlane(lane_ctx, b) : uniform(s_ctx[b]);
  };
  auto extents = [&](Fp4Unit& u) FP4_INLINE {
    fp4_extent<ROWS>(p, u.ctx, u.rb, &u.lo, &u.hi);
    u.first = fp4_first(u.lo);
    u.n = fp4_count(u.lo, u.hi);
  };
  // The last of 0 .. len - 1 with (s_pre[from + i stride] - s_pre[from]) mul <= key: 64 entries at a
  // time, one a lane.
  auto search = [&](int from, int len, int stride, int mul, int key) FP4_INLINE {
    int lo = 0;
    const int base = s_pre[from];
    while (len > 1) {
      const int step = (len + 63) >> 6;
      const int m = (lane + 1) * step;
      const bool le = m < len && (s_pre[from + (lo + m) * stride] - base) * mul <= key;
      const int c = __popcll(__ballot(le)) * step;
      lo += c;
      len = min(step, len - c);
    }
    return lo;
  };
  // The unit of the wave that holds position c0 of the list.
  Fp4Unit u{};
  int unit = 0;  // without a list: its number
  if constexpr (LIST) {
    u.b = regs ? __popcll(__ballot(lane < p.batch - 1 && lane_sum * p.KVH <= c0))
               : search(0, p.batch, p.rblocks, p.KVH, c0);
    const int e0 = u.b * p.rblocks;
    const int pre0 = sum_before(e0), per = sum_before(e0 + p.rblocks) - pre0;
    const int rem = c0 - pre0 * p.KVH;
    u.kvh = rem / per;
    const int in = rem - u.kvh * per;
    u.rb = p.rblocks == 1 ? 0 : search(e0, p.rblocks, 1, 1, in);
    u.u0 = pre0 * p.KVH + u.kvh * per + (sum_before(e0 + u.rb) - pre0) + kFp4Head;
    u.ctx = context(u.b);
    extents(u);
    u.skip = max(0, c0 - u.u0);
    u.cnt = min(u.n, c1 - u.u0) - u.skip;
  } else {
    // Without a list. Workgroup i runs on XCD i % 8, each of which has an L2 of its own: an XCD takes
    // a run of units, so that the row blocks of a head, which read the same keys, share one. Later
    // row blocks first: under a causal mask they have the most keys.
    const int at = ((share & 7) * p.xcd_units + (share >> 3)) * NU + wu;
    if constexpr (PARTS) unit = fp4_quot(at, p.by_parts);
    else unit = at;
    const int bk = fp4_quot(unit, p.by_rb);
    const int b = fp4_quot(bk, p.by_kvh);
    if (b < p.batch) {  // (waves past the last unit go on to the barriers, with one of no groups)
      u.rb = p.rblocks - 1 - (unit - bk * p.rblocks);
      u.b = b;
      u.kvh = bk - b * p.KVH;
      u.ctx = context(b);
      extents(u);
    }
    u.cnt = u.n;
    if constexpr (PARTS) {
      // Parts of equal length; a unit of a round of the waves or less is the first part's.
      const int part = at - unit * p.parts, q = fp4_quot(u.n, p.by_parts), more = u.n - q * p.parts;
      if (u.n > kFp4Waves) {
        u.skip = part * q + min(part, more);
        u.cnt = q + (part < more ? 1 : 0);
      } else if (part > 0 || u.n == 0) {
        return;  // (the workgroup as one)
      }
    }
    c1 = u.cnt;
  }
  if (LIST && u.cnt <= 0) return;  // (a share of the head of a unit alone; the workgroup as one)
  const bool head = u.cnt < u.n;   // the first unit has other shares
  if (LIST && tid == 0) {
    s_first[0] = u.b; s_first[1] = u.kvh; s_first[2] = u.rb; s_first[3] = u.u0; s_first[4] = u.n;
  }
  // Whether the share goes on behind u, and the unit it goes on with.
  auto more = [&](const Fp4Unit& u) FP4_INLINE { return u.u0 + u.n + kFp4Head < c1; };
  auto advance = [&](Fp4Unit& u) FP4_INLINE {
    u.u0 += u.n + kFp4Head;
    u.r0 += u.cnt;
    if (++u.rb == p.rblocks) {
      u.rb = 0;
      if (++u.kvh == p.KVH) {
        u.kvh = 0;
        u.ctx = context(++u.b);
      }
    }
    extents(u);
    u.skip = 0;
    u.cnt = min(u.n, c1 - u.u0);
  };
  int groups = u.cnt;  // of the share
  if constexpr (LIST) {
    if (more(u)) {
      Fp4Unit v = u;
      do advance(v);
      while (more(v));
      groups = v.r0 + v.cnt;
    }
  }

  // ---- what a lane holds of a tile: fixed places, one register each ----
  uint32_t k_at[HV], ks_at[HV], v_at[HV], vs_at[HV];
  bool k_in[HV];  // dims past D: keys read at the tile's start, times zeros of the query
#pragma unroll
  for (int h = 0; h < HV; ++h) {
    const int dim = 128 * h + g * LD;
    k_in[h] = dim < p.D;
    k_at[h] = k_in[h] ? n * (p.D / 2) + dim / 2 : 0;
    ks_at[h] = 8 * p.D + (k_in[h] ? 16 * (dim / 32) + n : 0);
    const int o = DH == 128 ? 16 * h + n : n / 2;
    const bool in = 8 * o < p.D;
    v_at[h] = in ? 64 * o + 16 * g : 0;
    vs_at[h] = 8 * p.D + (in ? 16 * (o / 4) + 4 * g : 0);
  }
  struct Tile {  // a tile's keys and values, and the scales of the lane's
    kraw_t k[HV];
    uint32_t ks[HV];
    uint4 v[HV];
    uint32_t vs[HV];
  };
  typedef Tile Group[2];

  // The wave takes the share's groups wk + WK s. Places of the tiles of its 32 groups from s = base on:
  // lane i holds tile i's byte offset, and bit i of `holes` says that the table has none (the offset
  // is then one that can be read). The table is asked first, and its answer taken up later.
  Fp4Unit ahead = u;  // the unit that the last places reached
  struct Asked {
    int page;      // as the table has it
    int64_t rest;  // the tile's bytes from its page's start on
  };
  auto ask = [&](int base) FP4_INLINE {
    const int r_first = wk + WK * base, r = r_first + WK * (lane >> 1);
    const int r_end = min(groups, r_first + WK * 32);
    int tile = 0, hi = 0;
    int64_t row = 0, head = 0;
    for (;;) {
      const int at = r - ahead.r0;
      if (at >= 0 && at < ahead.cnt) {
        tile = 2 * (ahead.first + ahead.skip + at) + (lane & 1);
        hi = ahead.hi;
        row = static_cast<int64_t>(ahead.b) * p.W;
        head = ahead.kvh * p.head_stride;
      }
      if (ahead.r0 + ahead.cnt >= r_end) break;
      advance(ahead);
    }
    Asked x;
    x.page = -1;
    const int pg = fp4_quot(tile, p.by_tiles);
    x.rest = head + static_cast<int64_t>(tile - pg * (p.bs / kFp4Tile)) * fp4_tile_bytes(p.D);
    if (tile * kFp4Tile < hi && pg < p.W) x.page = p.table[row + pg];
    return x;
  };
  auto answer = [&](const Asked& x, uint64_t* holes) FP4_INLINE {
    const bool has = x.page >= 0 && x.page < p.num_blocks;
    *holes = __ballot(!has);
    return has ? static_cast<int64_t>(x.page) * p.blk_stride + x.rest : int64_t(0);
  };
  uint64_t holes, next_holes = 0;
  int64_t here, next = 0;  // of this run of 32 groups, and of the next
  Asked asked{};           // of the next, until the run's last groups
  int run = 0;             // the run's first
  const int rounds = (groups - wk + WK - 1) / WK;  // groups of the wave
  // Keys (1), values (2) or both (3) of group s, of this run or the next, requested. Values alone come
  // after the same group's keys.
  int64_t at[2] = {0, 0};
  auto load = [&](Group& x, int s, auto parts_c) FP4_INLINE {
    constexpr int parts = decltype(parts_c)::value;
    if (s >= rounds) return;
    if constexpr ((parts & 1) != 0) {
      const int i = 2 * (s - run);
      auto from = [&](int64_t places, int t) FP4_INLINE {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(places), (i + t) & 63);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(places >> 32), (i + t) & 63);
        return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
      };
      if (i < 64) {  // (a branch: the next run's places may be on their way)
        at[0] = from(here, 0);
        at[1] = from(here, 1);
      } else {
        at[0] = from(next, 0);
        at[1] = from(next, 1);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const __amdgpu_buffer_rsrc_t kt = tile_rsrc(p.k + at[t], fp4_tile_bytes(p.D));
      const __amdgpu_buffer_rsrc_t vt = tile_rsrc(p.v + at[t], fp4_tile_bytes(p.D));
#pragma unroll
      for (int h = 0; h < HV; ++h) {
        if constexpr ((parts & 1) != 0) {
          x[t].k[h] = fp4_load<kraw_t>(kt, k_at[h]);
          x[t].ks[h] = fp4_load<uint8_t>(kt, ks_at[h]);
        }
        if constexpr ((parts & 2) != 0) {
          x[t].v[h] = fp4_load<uint4>(vt, v_at[h]);
          x[t].vs[h] = fp4_load<uint32_t>(vt, vs_at[h]);
        }
      }
    }
  };
  using Keys = std::integral_constant<int, 1>;
  using Values = std::integral_constant<int, 2>;
  using Both = std::integral_constant<int, 3>;

  // ---- a unit's state ----
  uint4 qf[QLDS ? 1 : CT][HV][NJ][PQ];
  static_assert(!QLDS || PQ == 1, "one part a query element");
  uint4* const s_q = reinterpret_cast<uint4*>(s_acc) + wu * (CT * HV * NJ * 64) + lane;
  mf_f32x4 acc[CT][HV][VC];
  float m_run[CT], l_run[CT];
  int lo_n[QLDS ? 1 : CT], hi_n[QLDS ? 1 : CT];  // keys the lane's rows see
  int all_lo, all_hi;      // keys every row of the block sees
  constexpr int QW = static_cast<int>(sizeof(T)) / 2;  // 16-byte words of 8 query elements
  uint4 q_raw[CT][HV][NJ][QW];
  auto query = [&]() FP4_INLINE {  // u's query rows, requested
    const int r0 = u.rb * ROWS;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int r = r0 + 16 * ct + n;
      const bool ok = r < p.rows_per_kvh;
      const int i = ok ? fp4_quot(r, p.by_g) : 0;
      const T* const qp = static_cast<const T*>(p.q) + u.b * p.q_st[0] + i * p.q_st[1] +
                          (u.kvh * p.G + (ok ? r - i * p.G : 0)) * p.q_st[2];
#pragma unroll
      for (int h = 0; h < HV; ++h)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int dim = 128 * h + g * LD + 8 * j;
#pragma unroll
          for (int x = 0; x < QW; ++x) {
            q_raw[ct][h][j][x] = make_uint4(0u, 0u, 0u, 0u);
            if (ok && dim < p.D)
              q_raw[ct][h][j][x] = *reinterpret_cast<const uint4*>(qp + dim + x * Chunk<T>::kElems);
          }
        }
    }
  };
  auto seen_keys = [&](const Fp4Unit& u, int r, int* lo, int* hi) FP4_INLINE {  // of row r of the KV head
    const int r1 = min(u.rb * ROWS + ROWS, p.rows_per_kvh) - 1;
    const int qpos = u.ctx - p.q_len + fp4_quot(min(r, r1), p.by_g);
    *hi = r > r1 ? 0 : (p.causal ? min(u.ctx, qpos + 1) : u.ctx);
    *lo = p.window > 0 ? max(0, qpos - p.window + 1) : 0;
  };
  auto begin = [&]() FP4_INLINE {
    const int ctx = u.ctx;
    const int r0 = u.rb * ROWS;
    const int r1 = min(r0 + ROWS, p.rows_per_kvh) - 1;
    const int q0 = ctx - p.q_len + fp4_quot(r0, p.by_g), q1 = ctx - p.q_len + fp4_quot(r1, p.by_g);
    all_hi = p.causal ? min(ctx, q0 + 1) : ctx;
    all_lo = p.window > 0 ? max(0, q1 - p.window + 1) : 0;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if constexpr (!QLDS) seen_keys(u, r0 + 16 * ct + n, &lo_n[ct], &hi_n[ct]);
      m_run[ct] = -INFINITY;
      l_run[ct] = 0.0f;
#pragma unroll
      for (int h = 0; h < HV; ++h) {
#pragma unroll
        for (int c = 0; c < VC; ++c) acc[ct][h][c] = mf_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if constexpr (QLDS) {  // (the unit's waves hold the same rows: one of them stores each)
            if ((ct * HV + h) * NJ + j == wk + ((ct * HV + h) * NJ + j) / WK * WK)
              s_q[((ct * HV + h) * NJ + j) * 64] = q_raw[ct][h][j][0];
          } else if constexpr (PQ == 1) {
            qf[ct][h][j][0] = q_raw[ct][h][j][0];
          } else {
            float x[8];
#pragma unroll
            for (int i = 0; i < QW; ++i)
              Chunk<T>::unpack(q_raw[ct][h][j][i], x + i * Chunk<T>::kElems);
#pragma unroll
            for (int a = 0; a < PQ; ++a) {
              const uint32_t w0 = fp4_cut2(x[0], x[1]), w1 = fp4_cut2(x[2], x[3]);
              const uint32_t w2 = fp4_cut2(x[4], x[5]), w3 = fp4_cut2(x[6], x[7]);
              qf[ct][h][j][a] = make_uint4(w0, w1, w2, w3);
            }
          }
        }
      }
    }
  };

  // Scores of the group's two tiles.
  auto scores = [&](const Group& x, mf_f32x4 (&s0)[CT], mf_f32x4 (&s1)[CT]) FP4_INLINE {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) s0[ct] = s1[ct] = mf_f32x4{0.f, 0.f, 0.f, 0.f};
    float sc[HV][2];
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int t = 0; t < 2; ++t) sc[h][t] = fp4_scale(k_in[h] ? x[t].ks[h] : 127u);
    // Word i of the 4 of step st (half st / NJ, product st % NJ) of tile t's operand.
    auto widen = [&](auto step_c, int t, int i) FP4_INLINE {
      constexpr int st = decltype(step_c)::value, h = st / NJ, j = st % NJ;
      const kraw_t& r = x[t].k[h];
      uint32_t w;
      if constexpr (DH == 128) w = j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w;
      else w = j == 0 ? r.x : r.y;
      return i == 0 ? fp4_widen2<0>(w, sc[h][t]) : i == 1 ? fp4_widen2<1>(w, sc[h][t])
             : i == 2 ? fp4_widen2<2>(w, sc[h][t]) : fp4_widen2<3>(w, sc[h][t]);
    };
    if constexpr (!QLDS) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        static_for<HV * NJ>([&](auto st_c) FP4_INLINE {
          constexpr int st = decltype(st_c)::value;
          const uint4 k = make_uint4(widen(st_c, t, 0), widen(st_c, t, 1), widen(st_c, t, 2), widen(st_c, t, 3));
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int a = 0; a < PQ; ++a) {
              mf_f32x4& s = t == 0 ? s0[ct] : s1[ct];
              s = Mfma16<bf16_t>::mac(k, qf[ct][st / NJ][st % NJ][a], s);
            }
        });
    } else {
      // One read of the query for both tiles, three of them on their way, and the keys of the next
      // step widened between the products of one (a wave issues in order).
      constexpr int kAhead = 3, kSteps = HV * NJ;
      uint32_t k[2][2][4];  // of the step's parity, by tile
      uint4 qv[kAhead];
      auto q_at = [&](int i) FP4_INLINE { return s_q[((i % CT * HV + i / CT / NJ) * NJ + i / CT % NJ) * 64]; };
#pragma unroll
      for (int i = 0; i < 8; ++i) k[0][i / 4][i % 4] = widen(std::integral_constant<int, 0>{}, i / 4, i % 4);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) qv[i] = q_at(i);
      static_for<kSteps>([&](auto st_c) FP4_INLINE {
        constexpr int st = decltype(st_c)::value;
        const uint4 k0 = make_uint4(k[st & 1][0][0], k[st & 1][0][1], k[st & 1][0][2], k[st & 1][0][3]);
        const uint4 k1 = make_uint4(k[st & 1][1][0], k[st & 1][1][1], k[st & 1][1][2], k[st & 1][1][3]);
        int i = 0;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int n = st * CT + ct;
          const uint4 q = qv[n % kAhead];
          s0[ct] = Mfma16<bf16_t>::mac(k0, q, s0[ct]);
          s1[ct] = Mfma16<bf16_t>::mac(k1, q, s1[ct]);
          if (n + kAhead < kSteps * CT) qv[n % kAhead] = q_at(n + kAhead);
          if constexpr (st + 1 < kSteps) {
#pragma unroll
            for (; i < 8 * (ct + 1) / CT; ++i)
              k[(st + 1) & 1][i / 4][i % 4] = widen(std::integral_constant<int, st + 1>{}, i / 4, i % 4);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      });
    }
  };

  uint4 pw[CT][PW];  // the weights, as the B operand of the value products
  float psum[CT];
  auto weights = [&](int ct, const mf_f32x4& s0, const mf_f32x4& s1, float mul) FP4_INLINE {
    const float m = m_run[ct] != -INFINITY ? m_run[ct] : 0.0f;
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = __builtin_amdgcn_exp2f(fmaf(s0[i], mul, -m));
      x[4 + i] = __builtin_amdgcn_exp2f(fmaf(s1[i], mul, -m));
    }
    psum[ct] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
    for (int a = 0; a < PW; ++a) {
      const uint32_t w0 = fp4_part2(x[0], x[1]), w1 = fp4_part2(x[2], x[3]);
      const uint32_t w2 = fp4_part2(x[4], x[5]), w3 = fp4_part2(x[6], x[7]);
      pw[ct][a] = make_uint4(w0, w1, w2, w3);
    }
  };
  // The weights with the running maximum as it stands, and only where one of them exceeds 2^8 (or
  // the row has no maximum yet) with one that has moved: their sum bounds each of them.
  auto softmax = [&](const mf_f32x4 (&s0)[CT], const mf_f32x4 (&s1)[CT], float mul) FP4_INLINE {
    bool over = false;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      weights(ct, s0[ct], s1[ct], mul);
      over = over || psum[ct] > 256.0f || m_run[ct] == -INFINITY;
    }
    if (__builtin_expect(__any(over), 0)) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float t = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) t = fmaxf(t, fmaxf(s0[ct][i] * mul, s1[ct][i] * mul));
        t = rows4_max(t);
        const float m = fmaxf(m_run[ct], t);
        const float alpha = m != -INFINITY ? __builtin_amdgcn_exp2f(m_run[ct] - m) : 1.0f;
        m_run[ct] = m;
        l_run[ct] *= alpha;
#pragma unroll
        for (int h = 0; h < HV; ++h)
#pragma unroll
          for (int c = 0; c < VC; ++c) acc[ct][h][c] *= alpha;
        weights(ct, s0[ct], s1[ct], mul);
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) l_run[ct] += psum[ct];
  };

  // O^T += V^T P^T for half h: d0, d1 the tiles' elements, sc the 8 tokens' scales.
  auto product = [&](auto h_c, const uint4& d0, const uint4& d1, const float (&sc)[8],
                     const uint4 (&b)[CT][PW]) FP4_INLINE {
    constexpr int h = decltype(h_c)::value;
    uint32_t x[8] = {d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
    if constexpr (DH == 64) {  // two lanes share 8 dims
      const int sh = 16 * (n & 1);
#pragma unroll
      for (int t = 0; t < 8; ++t) x[t] >>= sh;
    }
    // The operands of dims 2 c and 2 c + 1, widened step by step between the products of the two dims
    // before (a wave issues in order: the matrix core runs while it widens).
    uint32_t e[2][4], o[2][4], y[2];
    auto step = [&](auto c_c, int t) FP4_INLINE {
      constexpr int c = decltype(c_c)::value;
      y[t & 1] = fp4_widen2<c>(x[t], sc[t]);
      if (t & 1) {
        e[c & 1][t / 2] = __builtin_amdgcn_perm(y[1], y[0], 0x05040100u);
        o[c & 1][t / 2] = __builtin_amdgcn_perm(y[1], y[0], 0x07060302u);
      }
    };
#pragma unroll
    for (int t = 0; t < 8; ++t) step(std::integral_constant<int, 0>{}, t);
    static_for<VC / 2>([&](auto cc) FP4_INLINE {
      constexpr int c = decltype(cc)::value;
      const uint4 ea = make_uint4(e[c & 1][0], e[c & 1][1], e[c & 1][2], e[c & 1][3]);
      const uint4 oa = make_uint4(o[c & 1][0], o[c & 1][1], o[c & 1][2], o[c & 1][3]);
      constexpr int N = CT * PW;  // pairs of products
      int t = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ct = i / PW, a = i % PW;
        acc[ct][h][2 * c] = Mfma16<bf16_t>::mac(ea, b[ct][a], acc[ct][h][2 * c]);
        acc[ct][h][2 * c + 1] = Mfma16<bf16_t>::mac(oa, b[ct][a], acc[ct][h][2 * c + 1]);
        if constexpr (c + 1 < VC / 2) {
#pragma unroll
          for (; t < 8 * (i + 1) / N; ++t) step(std::integral_constant<int, c + 1>{}, t);
        }
        if constexpr (CT > 1) __builtin_amdgcn_sched_barrier(0);
      }
    });
  };
  auto byte_of = [](uint32_t x, int i) { return (x >> (8 * i)) & 255u; };

  auto consume = [&](Group& x, int s) FP4_INLINE {
    const int tok = (u.first + u.skip + wk + WK * s - u.r0) * kFp4Group;
    mf_f32x4 s0[CT], s1[CT];
    scores(x, s0, s1);
    if constexpr (kEarly) load(x, s + kRing, Keys{});  // (the keys' registers are free)
    const uint32_t hole = static_cast<uint32_t>(holes >> (2 * (s - run))) & 3u;
    const bool full = tok >= all_lo && tok + kFp4Group <= all_hi && hole == 0;
    float mul = p.scale_log2;
    // Of keys 4 g + i of tile t, bit 4 t + i: where the lane's row sees them, and where a value's
    // block is NaN (in groups that have masked keys).
    uint32_t seen[CT], bad[HV], any_bad = 0;
    if (!full) {
      uint32_t dead = 0;  // no row sees it, or the table has no page
      int lo_r[CT], hi_r[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        seen[ct] = 0;
        if constexpr (QLDS) {  // (worked out here: the registers are the accumulators')
          uint32_t row = u.rb * ROWS + 16 * ct + n;
          opaque(row);
          seen_keys(u, static_cast<int>(row), &lo_r[ct], &hi_r[ct]);
        } else {
          lo_r[ct] = lo_n[ct];
          hi_r[ct] = hi_n[ct];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = tok + 16 * (i / 4) + 4 * g + i % 4;
        const bool live = key >= u.lo && key < u.hi && !((hole >> (i / 4)) & 1u);
        dead |= live ? 0u : 1u << i;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const bool see = live && key >= lo_r[ct] && key < hi_r[ct];
          seen[ct] |= see ? 1u << i : 0u;
          // (scaled first: a scale of 0 or below must not touch the mask)
          if (i < 4) s0[ct][i % 4] = see ? s0[ct][i % 4] * p.scale_log2 : -INFINITY;
          else s1[ct][i % 4] = see ? s1[ct][i % 4] * p.scale_log2 : -INFINITY;
        }
      }
      mul = 1.0f;
#pragma unroll
      for (int h = 0; h < HV; ++h) {
        bad[h] = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint32_t e[4] = {x[t].v[h].x, x[t].v[h].y, x[t].v[h].z, x[t].v[h].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool gone = (dead >> (4 * t + i)) & 1u;
            const bool nan = byte_of(x[t].vs[h], i) == kFp4NaN;
            bad[h] |= nan && !gone ? 1u << (4 * t + i) : 0u;
            e[i] = gone || nan ? 0u : e[i];
            x[t].vs[h] = gone || nan ? (x[t].vs[h] & ~(255u << (8 * i))) | 127u << (8 * i)
                                       : x[t].vs[h];
          }
          x[t].v[h] = make_uint4(e[0], e[1], e[2], e[3]);
        }
        any_bad |= bad[h];
      }
    }
    softmax(s0, s1, mul);
    static_for<HV>([&](auto hc) FP4_INLINE {
      constexpr int h = decltype(hc)::value;
      float sc[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[i] = fp4_scale_of(x[0].vs[h], i);
        sc[4 + i] = fp4_scale_of(x[1].vs[h], i);
      }
      product(hc, x[0].v[h], x[1].v[h], sc, pw);
    });
    if (!full && __any(any_bad != 0)) {
      // Rows that see a NaN block of dims: ones for the blocks times ones for what the rows see.
      auto ones = [](uint32_t bits) FP4_INLINE {
        opaque(bits);  // (else the compiler works these out for every group)
        uint32_t y[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          y[t] = ((bits >> (2 * t)) & 1u ? 0x3f80u : 0u) | ((bits >> (2 * t + 1)) & 1u ? 0x3f800000u : 0u);
        return make_uint4(y[0], y[1], y[2], y[3]);
      };
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int h = 0; h < HV; ++h) {
          const mf_f32x4 hit =
              Mfma16<bf16_t>::mac(ones(bad[h]), ones(seen[ct]), mf_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[ct][h][c][i] = hit[i] > 0.0f ? __uint_as_float(0x7fc00000u) : acc[ct][h][c][i];
        }
    }
  };

  auto out_at = [&](const Fp4Unit& u, int r) FP4_INLINE {  // element offset of row r of the unit's KV head in the output
    const int i = fp4_quot(r, p.by_g);
    return ((static_cast<int64_t>(u.b) * p.q_len + i) * p.H + (u.kvh * p.G + (r - i * p.G))) * p.D;
  };
  // The waves' parts of unit u joined, 16 rows at a time: normalised rows, or the share's partial.
  // At the share's end all threads do it, between barriers. Before, a wave leaves its part in a
  // buffer and goes on to the next unit, and the last to leave one joins them: no wave waits for the
  // others, unless all buffers hold parts of earlier units.
  const int brows = LIST ? min(16, p.slot_rows) : 16, buffers = 16 / brows;
  int event = 0;
  auto put = [&](int ct, int buf, int rows) FP4_INLINE {
    const float l = rows4_sum(l_run[ct]);
    if (n >= rows) return;
    const int at = (buf * kFp4Waves + w) * brows + n;
    if (g == 0) s_ml[at] = make_float2(m_run[ct], l);
#pragma unroll
    for (int h = 0; h < HV; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < VC; c += 4)
          *reinterpret_cast<float4*>(&s_acc[at * RS + 128 * h + LD * g + VC * i + c]) =
              make_float4(acc[ct][h][c][i], acc[ct][h][c + 1][i], acc[ct][h][c + 2][i],
                          acc[ct][h][c + 3][i]);
  };
  auto fold = [&](const Fp4Unit& u, int r0, int buf, int rows, int t0, int threads) FP4_INLINE {
    const int per = p.D / 4;  // items of a row
    const bool whole = u.cnt == u.n;
    const int64_t slot = PARTS ? static_cast<int64_t>((share & 7) * p.xcd_units + (share >> 3))
                               : 2 * static_cast<int64_t>(share) + (u.skip == 0 ? 1 : 0);
    for (int idx = t0; idx < rows * per; idx += threads) {
      const int r = fp4_quot(idx, p.by_per), d = 4 * (idx - r * per);
      float2 ml[WK];
      float M = -INFINITY, L = 0.0f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      const int at = buf * brows + r;  // (buf: the first wave's part)
#pragma unroll
      for (int i = 0; i < WK; ++i) {
        ml[i] = s_ml[at + i * brows];
        M = fmaxf(M, ml[i].x);
      }
#pragma unroll
      for (int i = 0; i < WK; ++i) {
        const float f = __builtin_amdgcn_exp2f(M != -INFINITY ? ml[i].x - M : 0.0f);
        const float4 x = *reinterpret_cast<const float4*>(&s_acc[(at + i * brows) * RS + d]);
        L = fmaf(f, ml[i].y, L);
        a.x = fmaf(f, x.x, a.x);
        a.y = fmaf(f, x.y, a.y);
        a.z = fmaf(f, x.z, a.z);
        a.w = fmaf(f, x.w, a.w);
      }
      if (whole) {
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;  // (a NaN stays one)
        fp4_store4<T>(static_cast<T*>(p.out) + out_at(u, u.rb * ROWS + r0 + r) + d, a.x * inv,
                      a.y * inv, a.z * inv, a.w * inv);
      } else {
        const int64_t row = slot * p.slot_rows + r0 + r;
        if (d == 0) store2_device(p.ml + row * 2, M, L);
        store2_device(p.acc + row * p.D + d, a.x, a.y);
        store2_device(p.acc + row * p.D + d + 2, a.z, a.w);
      }
    }
  };
  auto finish = [&](const Fp4Unit& u, bool ends) FP4_INLINE {
    const int rows = u.n == 0 ? 0 : min(ROWS, p.rows_per_kvh - u.rb * ROWS);  // (no unit: none)
    if (ends) {
      lds_barrier();  // (the buffers' last parts are read)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int n_rows = min(16, rows - 16 * ct);  // (units of one workgroup may differ)
        if (NU == 1 && n_rows <= 0) break;
        put(ct, 0, n_rows);
        lds_barrier();
        fold(u, 16 * ct, wu * WK, n_rows, tid - 64 * WK * wu, 64 * WK);
        lds_barrier();
      }
      return;
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int n_rows = min(16, rows - 16 * ct);
      if (n_rows <= 0) break;
      const int gen = event / buffers, buf = event - gen * buffers;
      ++event;
      // (every wave leaves its part of each event in turn, so that the one waited for comes)
      while (__hip_atomic_load(&s_done[buf], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) < gen)
        __builtin_amdgcn_s_sleep(1);
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      put(ct, buf, n_rows);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      int old = 0;
      if (lane == 0)
        old = __hip_atomic_fetch_add(&s_cnt[buf], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      old = uniform(old);
      if (old != kFp4Waves * gen + kFp4Waves - 1) continue;
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      fold(u, 16 * ct, buf * kFp4Waves, n_rows, lane, 64);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
      if (lane == 0)
        __hip_atomic_store(&s_done[buf], gen + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  };
  // The join of unit v, whose shares have all left their partials.
  auto join = [&](const Fp4Unit& v) FP4_INLINE {
    const int r0 = v.rb * ROWS;
    const int rows = min(ROWS, p.rows_per_kvh - r0);
    const int per = p.D / 4;
    const int s_first = PARTS ? unit * p.parts : v.u0 / chunk;
    const int s_last = PARTS ? s_first + p.parts - 1 : (v.u0 + v.n - 1) / chunk;
    // Threads left over take other shares of the same items, and are joined through LDS.
    const int items = rows * per;
    const int parts = items >= kFp4Threads ? 1 : kFp4Threads / items;
    float* const s_part = s_acc;  // [thread][6]
    for (int i0 = 0; i0 < items; i0 += kFp4Threads) {
      const int k = parts == 1 ? 0 : tid / items;
      const int idx = parts == 1 ? i0 + tid : tid - k * items;
      const bool mine = idx < items && k < parts;
      const int r = mine ? fp4_quot(idx, p.by_per) : 0, d = mine ? 4 * (idx - r * per) : 0;
      float M = -INFINITY, L = 0.0f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      constexpr int N = 4;
      for (int j0 = s_first + k; mine && j0 <= s_last; j0 += N * parts) {
        float2 x0[N], x1[N], ml[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {  // shares past the last repeat it, unused
          const int j = min(j0 + i * parts, s_last);
          const int64_t slot = PARTS ? j : 2 * static_cast<int64_t>(j) + (j == s_first ? 1 : 0);
          const int64_t row = slot * p.slot_rows + r;
          ml[i] = load2_device(p.ml + row * 2);
          x0[i] = load2_device(p.acc + row * p.D + d);
          x1[i] = load2_device(p.acc + row * p.D + d + 2);
        }
        float mb = M;
#pragma unroll
        for (int i = 0; i < N; ++i) mb = fmaxf(mb, j0 + i * parts <= s_last ? ml[i].x : -INFINITY);
        const float keep = __builtin_amdgcn_exp2f(mb != -INFINITY ? M - mb : 0.0f);
        L *= keep;
        a.x *= keep; a.y *= keep; a.z *= keep; a.w *= keep;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool live = j0 + i * parts <= s_last;
          const float f = __builtin_amdgcn_exp2f(live && mb != -INFINITY ? ml[i].x - mb : 0.0f);
          L = live ? fmaf(f, ml[i].y, L) : L;
          a.x = live ? fmaf(f, x0[i].x, a.x) : a.x;
          a.y = live ? fmaf(f, x0[i].y, a.y) : a.y;
          a.z = live ? fmaf(f, x1[i].x, a.z) : a.z;
          a.w = live ? fmaf(f, x1[i].y, a.w) : a.w;
        }
        M = mb;
      }
      if (parts > 1) {
        float* const mine_at = s_part + 6 * tid;
        mine_at[0] = M; mine_at[1] = L; mine_at[2] = a.x; mine_at[3] = a.y; mine_at[4] = a.z;
        mine_at[5] = a.w;
        lds_barrier();
        if (mine && k == 0) {
          float mb = M;
          for (int i = 1; i < parts; ++i) mb = fmaxf(mb, s_part[6 * (tid + i * items)]);
          const float keep = __builtin_amdgcn_exp2f(mb != -INFINITY ? M - mb : 0.0f);
          L *= keep;
          a.x *= keep; a.y *= keep; a.z *= keep; a.w *= keep;
          for (int i = 1; i < parts; ++i) {
            const float* const x = s_part + 6 * (tid + i * items);
            const float f = __builtin_amdgcn_exp2f(mb != -INFINITY ? x[0] - mb : 0.0f);
            L = fmaf(f, x[1], L);
            a.x = fmaf(f, x[2], a.x);
            a.y = fmaf(f, x[3], a.y);
            a.z = fmaf(f, x[4], a.z);
            a.w = fmaf(f, x[5], a.w);
          }
        }
        lds_barrier();
      }
      if (mine && k == 0) {
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;
        fp4_store4<T>(static_cast<T*>(p.out) + out_at(v, r0 + r) + d, a.x * inv, a.y * inv, a.z * inv,
                      a.w * inv);
      }
    }
  };

  // ---- the share ----
  asked = ask(0);
  query();
  here = answer(asked, &holes);
  Group ring[kRing];  // the next groups, on their way
  static_for<kRing>([&](auto i) FP4_INLINE { load(ring[i], i, Both{}); });
  if (rounds > 32) asked = ask(32);
  lds_barrier();  // (the counters are set)
  int s = 0, turn = 0;  // the wave's next group, and where in the ring it is
  for (;;) {
    begin();
    if constexpr (QLDS) lds_barrier();  // (units of their own: each wave comes here once)
    const int s_end = (u.r0 + u.cnt - wk + WK - 1) / WK;
    for (; s < s_end; ++s) {
      if (s - run == 32 - kRing) next = answer(asked, &next_holes);
      if (s - run == 32) {
        run = s;
        here = next;
        holes = next_holes;
        if (rounds > s + 32) asked = ask(s + 32);
      }
      // (a copy of the code for each place of the ring: its registers are not moved)
      static_for<kRing>([&](auto i) FP4_INLINE {
        if (turn == i) {
          consume(ring[i], s);
          load(ring[i], s + kRing, typename std::conditional<kEarly, Values, Both>::type{});
        }
      });
      turn = turn == kRing - 1 ? 0 : turn + 1;
      if (WK == kFp4Waves && CT == 1 && (s & 1) == 0) {
        // Of a SIMD's two waves the older one's loads are served first: the one that is not ahead
        // issues at a raised priority.
        __hip_atomic_store(&s_prog[w], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        const int other = uniform(__hip_atomic_load(&s_prog[w ^ 4], __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_WORKGROUP));
        if (s <= other) __builtin_amdgcn_s_setprio(1);
        else __builtin_amdgcn_s_setprio(0);
      }
    }
    if constexpr (!LIST) {
      finish(u, true);
      break;
    }
    const Fp4Unit done = u;
    const bool go_on = more(u);
    if (go_on) {
      advance(u);
      query();
    }
    finish(done, !go_on);
    if (!go_on) break;
  }

  if constexpr (WAY == kFp4Dealt) return;
  if constexpr (PARTS) {
    if (u.cnt == u.n) return;
    // (as below, with a counter a unit)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (tid == 0) {
      int* const t = p.tickets + unit;
      const int old = __hip_atomic_fetch_add(t, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      const bool last = old == p.parts - 1;
      if (last) __hip_atomic_store(t, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      s_tot[0] = last;
    }
    lds_barrier();
    const int last = uniform(s_tot[0]);
    asm volatile("" ::: "memory");
    if (last) join(u);
    return;
  }
  // ---- the first and the last unit, where they have other shares ----
  const bool tail = u.cnt < u.n;  // (u: the last; perhaps the first too)
  if (!head && !tail) return;
  // The partials are written through (agent scope) before the counters move, and read the same way
  // after them. A unit's counter is its first share's, which no other unit split has.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  lds_barrier();
  Fp4Unit first{};
  first.b = uniform(s_first[0]);
  first.kvh = uniform(s_first[1]);
  first.rb = uniform(s_first[2]);
  first.u0 = uniform(s_first[3]);
  first.n = uniform(s_first[4]);
  if (tid < 2) {
    const Fp4Unit& v = tid == 0 ? first : u;
    const int mine = tid == 0 ? head && first.u0 != u.u0 : tail;
    int last = 0;
    if (mine) {
      const int s_first = v.u0 / chunk, s_last = (v.u0 + v.n - 1) / chunk;
      int* const t = p.tickets + s_first;
      const int old = __hip_atomic_fetch_add(t, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = old == s_last - s_first;
      if (last) __hip_atomic_store(t, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    s_tot[tid] = last;
  }
  lds_barrier();
  const int last0 = uniform(s_tot[0]), last1 = uniform(s_tot[1]);
  asm volatile("" ::: "memory");
  for (int i = 0; i < 2; ++i) {
    if (i == 0 ? last0 : last1) join(i == 0 ? first : u);
  }
}

// Blocks of 16 query rows that a wave takes at most, by the bf16 parts of a query element: what its
// registers hold of accumulators, query and the groups on their way. Past it they spill: at 256 dims two
// blocks 500 bytes a lane and more (40 rows of 4 drafts of H8/KVH1, 300 to 2000 keys, as units of eight
// waves: 99 us against 25), fp32 of 128 dims 150 (2 x 512 queries of H28/KVH4 behind 4096 keys, units of
// two waves: 205 against 191).
constexpr int fp4_max_ct(int parts, int DP) {
  return DP > 128 || (DP > 64 && parts == 3) ? 1 : (parts == 1 ? 4 : 2);
}
// Of a list, whose kernel holds more besides (two blocks of fp16 of 128 dims 270 bytes: 32 rows of 4 drafts
// of H28/KVH4, 600 to 4096 keys, 60 us against 30).
constexpr int fp4_list_ct(int parts, int DP) { return DP > 128 || (DP > 64 && parts > 1) ? 1 : 2; }

template <typename T, int DP>
hipError_t launch_fp4_attn(const Fp4Params& p, int way, int ct, int wk, hipStream_t stream);

}  // namespace msattn
