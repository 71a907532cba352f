// Attention for a batch whose rows come in groups, each group behind a prefix of its own: the
// same physical pages in every row of the group (gfx950; a bf16/fp16 query over a cache of its
// type or of fp8 e4m3, head_dim 64 or 128, any number of query tokens a row).
//
// The work is a list of segments: one a group (the prefix's keys, read once for the query rows of
// every member) and one a batch row (the keys past its prefix, or all of them). A segment falls
// into units, one a KV head and block of up to 128 query rows; a unit's keys are cut into tiles
// of 128. All tiles of all units, in order, are dealt in equal contiguous shares, one a
// workgroup, whatever the lengths (they are read on the device, so a call is capture-safe). A
// share's part of one unit is a piece; it leaves, for each of its query rows,
//   m = max_j s_j,  l = sum_j 2^(s_j - m),  acc = sum_j 2^(s_j - m) V_j,   s_j = scale log2(e) q.K_j
// over the piece's visible keys, and the merge kernel below joins a row's pieces:
//   out = sum 2^(m - M) acc / sum 2^(m - M) l,   M = max m.
//
// A tile's 16 KB to 32 KB each of K and V are copied into LDS by the load unit, two tiles in
// flight while one is computed, across piece and unit boundaries, so the memory pipe does not run
// dry between units. Scores are S^T = K Q^T on v_mfma_f32_16x16x32, 16 query rows a wave: lane
// (g, n) = (l / 16, l % 16) then holds row n's scores of keys 4 g .. 4 g + 3 of a 16-key block,
// and two such blocks, rounded to the query type and packed, are its B operand of
// O^T += V^T P^T (V^T by transposed LDS reads), so softmax and rescaling stay in the lane.
// A unit of more than 64 query rows gives each of the 8 waves 16 rows and all keys; fewer rows
// leave waves over, which take every second or fourth 32-key block of the same rows and are
// joined through LDS at the piece's end.
//
// Semantics: miniserve/attention.py:205-250 (causal), whose gather reads a shared page once a row.
#pragma once

#include "prefill_mfma.h"

namespace msattn {

constexpr int kShWaves = 8;
constexpr int kShThreads = kShWaves * kWave;
constexpr int kShTile = 16 * kShWaves;  // keys of a tile: 16 a copying wave
constexpr int kShRows = 16 * kShWaves;  // query rows of a unit, at most
constexpr int kShMaxBatch = 1024;       // rows (and groups) of a launch: its plan sits in LDS
constexpr int kShIds = kWave;           // page ids a wave holds: its sub-tile's in 64 tiles

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
  int bs, bs_shift, num_blocks, W, max_ctx;
  float scale_log2;
  // Workspace: the plan (written by workgroup 0 for the merge) and the pieces' partials. A
  // unit's first piece goes to slot kind * rows + output row (kind 0: the group's segment, 1: the
  // row's own), a later one to slot 2 * rows + share * kShRows + row of the unit.
  int* plan;   // [0] tiles a share, [kShPlanCum ..] tiles before each segment, then group ids
  float* ml;   // [slots][2]
  float* acc;  // [slots][D]
  int64_t rows;  // batch * q_len * H
  int shares;
};

constexpr int kShPlanCum = 16;
__host__ __device__ constexpr int sh_plan_words(int batch, int groups) {
  return kShPlanCum + (groups + batch + 1) + batch + (groups + 1);
}
__host__ __device__ constexpr int64_t sh_slots(int64_t rows, int shares) {
  return 2 * rows + static_cast<int64_t>(shares) * kShRows;
}

// s_waitcnt immediates (gfx9 encoding): at most N vector memory operations outstanding.
constexpr int sh_wait_vm(int n) { return 0x0F70 | (n & 15); }

template <typename T, typename KT, int D>
__global__ __launch_bounds__(kShThreads, 2) void shared_attn_kernel(
    const SharedParams p) {
  typedef Kv8<T, KT> KV;
  static_assert(D == 64 || D == 128, "head_dim 64 and 128");
  constexpr int EB = static_cast<int>(sizeof(KT));
  constexpr bool WIDEN = !std::is_same<T, KT>::value;  // fp8 rows pass through registers
  constexpr int JD = D / 32;  // MFMA k-steps of a score block
  constexpr int ND = D / 16;  // 16-dim tiles of O^T
  constexpr int CPR = D * EB / 16;   // 16-byte chunks a cache row
  constexpr int RPI = kWave / CPR;   // rows a copy instruction
  constexpr int NI = 16 / RPI;       // copy instructions a 16-row sub-tile

  __shared__ __attribute__((aligned(256))) uint16_t s_k0[kShTile * D];
  __shared__ __attribute__((aligned(256))) uint16_t s_v0[kShTile * D];
  __shared__ __attribute__((aligned(256))) uint16_t s_k1[kShTile * D];
  __shared__ __attribute__((aligned(256))) uint16_t s_v1[kShTile * D];
  __shared__ int s_cum[2 * kShMaxBatch + 1];  // tiles before each segment: groups, then rows
  __shared__ int s_g0[kShMaxBatch + 1];       // a group's first row
  __shared__ int s_hi[kShMaxBatch];           // a group's last visible prefix key + 1
  __shared__ int s_len[kShMaxBatch];
  __shared__ int s_own[kShMaxBatch];          // where a row's own keys begin
  __shared__ float2 s_ml[kShWaves][16];
  __shared__ int s_live[2][kShWaves];         // sub-tiles of the two tiles that are no holes
  __shared__ int s_wsum[kShWaves];

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int w = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int g = lane >> 4;
  const int n = lane & 15;
  const int B = p.batch, NG = p.groups, NS = NG + B;
  const int RPS = p.q_len * p.G;  // query rows a KV head and batch row

  // ---- the plan: tiles before each segment ----
  for (int i = tid; i <= NG; i += kShThreads) {
    const int r = NG > 0 ? p.group_rows[i] : 0;
    s_g0[i] = r < 0 ? 0 : (r > B ? B : r);
    if (i < NG) s_hi[i] = 0;
  }
  for (int b = tid; b < B; b += kShThreads) {
    const int len = p.lens[b];
    s_len[b] = len < 0 ? 0 : (len > p.max_ctx ? p.max_ctx : len);
  }
  __syncthreads();
  const int own_rtiles = ceil_div(RPS, kShRows);
  for (int b = tid; b < B; b += kShThreads) {
    int lo = 0, hi = NG;  // the last group that begins at or before row b
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_g0[mid] <= b) lo = mid; else hi = mid;
    }
    int own = 0, grp = -1;
    // (a group of one row has nothing to share: its prefix is the row's own)
    if (NG > 0 && s_g0[lo] <= b && b < s_g0[lo + 1] && s_g0[lo + 1] - s_g0[lo] > 1) {
      int pages = p.prefix_pages[lo];
      pages = pages < 0 ? 0 : (pages > p.W ? p.W : pages);
      const int64_t pt = static_cast<int64_t>(pages) * p.bs;
      own = static_cast<int>(pt < p.max_ctx ? pt : p.max_ctx);
      grp = lo;
      atomicMax(&s_hi[lo], min(own, s_len[b]));
    }
    s_own[b] = own;
    s_cum[NG + b] = s_len[b] > own ? ceil_div(s_len[b] - own, kShTile) * p.KVH * own_rtiles : 0;
    if (blockIdx.x == 0) p.plan[kShPlanCum + NS + 1 + b] = grp;
  }
  __syncthreads();
  for (int i = tid; i < NG; i += kShThreads)
    s_cum[i] = ceil_div(s_hi[i], kShTile) * p.KVH *
               ceil_div(max(0, s_g0[i + 1] - s_g0[i]) * RPS, kShRows);
  __syncthreads();
  {
    constexpr int kPer = 2 * kShMaxBatch / kShThreads;
    int c[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = tid * kPer + i;
      c[i] = e < NS ? s_cum[e] : 0;
      sum += c[i];
    }
    const int incl = wave_inclusive_sum(sum);
    if (lane == kWave - 1) s_wsum[w] = incl;
    __syncthreads();
    int at = incl - sum;
    for (int i = 0; i < w; ++i) at += s_wsum[i];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = tid * kPer + i;
      if (e < NS) s_cum[e] = at;
      at += c[i];
      if (e == NS - 1) s_cum[NS] = at;
    }
    __syncthreads();
  }
  const int total = __builtin_amdgcn_readfirstlane(s_cum[NS]);
  const int per = max(1, ceil_div(total, p.shares));
  if (blockIdx.x == 0) {
    if (tid == 0) p.plan[0] = per;
    for (int i = tid; i <= NS; i += kShThreads) p.plan[kShPlanCum + i] = s_cum[i];
    for (int i = tid; i <= NG; i += kShThreads) p.plan[kShPlanCum + NS + 1 + B + i] = s_g0[i];
  }
  // Contiguous shares to one XCD (workgroup i runs on XCD i % 8): the row blocks of one KV head
  // then read their keys through one L2.
  const int share = p.shares % kXcds == 0
                        ? static_cast<int>(blockIdx.x % kXcds) * (p.shares / kXcds) +
                              static_cast<int>(blockIdx.x / kXcds)
                        : static_cast<int>(blockIdx.x);
  const int64_t first64 = static_cast<int64_t>(share) * per;
  if (first64 >= total) return;
  const int first = static_cast<int>(first64);
  const int last = min(total, first + per);

  // A piece: tiles t0 .. t1 - 1 of one unit.
  struct Piece {
    int kind;         // 0: a group's segment, 1: a row's own
    int b0;           // the batch row whose table names the pages, and the segment's first row
    int kvh, row0, nrows;  // query rows row0 .. row0 + nrows - 1 of the segment, for one KV head
    int key0, hi;     // the segment's keys are key0 .. hi - 1
    int t0, t1;
  };
  const auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  auto locate = [&](int pos) __attribute__((always_inline)) {
    int lo = 0, hi = NS;  // the last segment that begins at or before pos
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (uni(s_cum[mid]) <= pos) lo = mid; else hi = mid;
    }
    Piece c;
    int members = 1;
    if (lo < NG) {
      c.kind = 0;
      c.b0 = uni(s_g0[lo]);
      members = uni(s_g0[lo + 1]) - c.b0;
      c.key0 = 0;
      c.hi = uni(s_hi[lo]);
    } else {
      c.kind = 1;
      c.b0 = lo - NG;
      c.key0 = uni(s_own[c.b0]);
      c.hi = uni(s_len[c.b0]);
    }
    const int tiles = ceil_div(c.hi - c.key0, kShTile);
    const int off = pos - uni(s_cum[lo]);
    const int unit = off / tiles;
    const int rtiles = ceil_div(members * RPS, kShRows);
    c.kvh = unit / rtiles;
    c.row0 = (unit - c.kvh * rtiles) * kShRows;
    c.nrows = min(kShRows, members * RPS - c.row0);
    c.t0 = off - unit * tiles;
    c.t1 = min(tiles, c.t0 + (last - pos));
    return c;
  };

  // ---- copying: wave w takes keys 16 w .. 16 w + 15 of each tile ----
  const KT* const kbase = static_cast<const KT*>(p.k);
  const KT* const vbase = static_cast<const KT*>(p.v);
  const int64_t row_bytes = p.slot_stride * EB;
  uint32_t dvo[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int lr = RPI * j + lane / CPR;
    dvo[j] = static_cast<uint32_t>(lr * row_bytes +
                                   16 * (WIDEN ? lane % CPR : (lane % CPR) ^ pf_swz<D>(lr)));
  }
  auto page_of = [&](int tok) { return p.bs_shift >= 0 ? tok >> p.bs_shift : tok / p.bs; };
  // Lane i: the page id of this wave's sub-tile in tile t + i of the piece (-1: none).
  auto load_ids = [&](const Piece& c, int t) __attribute__((always_inline)) {
    const int64_t tok = c.key0 + static_cast<int64_t>(t + lane) * kShTile + 16 * w;
    int id = -1;
    if (t + lane < c.t1 && tok < c.hi) {
      const int pg = page_of(static_cast<int>(tok));
      if (pg < p.W) id = p.table[static_cast<int64_t>(c.b0) * p.W + pg];
    }
    return id;
  };

  // The copying cursor runs two tiles ahead of the computing one.
  Piece lp = locate(first);
  int lpos = first, lt = lp.t0, lw = lp.t0;  // tile lt, its piece, the first tile of the ids held
  int ids = load_ids(lp, lw);
  constexpr int HOLD = WIDEN ? 2 : 1;  // fp8: two tiles are held in registers
  uint4 k_held[HOLD][NI], v_held[HOLD][NI];
  int live_held[HOLD];
  // Requests tile lpos into slot `buf` (fp8: into register set `buf`, which land() widens into
  // the slot), and moves the cursor on. The page ids of a new piece or window are requested
  // first, so that the next tile waits for them alone.
  auto request = [&](uint16_t* sk, uint16_t* sv, int buf, auto set_c) __attribute__((always_inline)) {
    constexpr int set = decltype(set_c)::value;
    const bool live = lpos < last;
    int phys = -1, tok = 0, kvh = 0, hi = 0;
    if (live) {
      phys = __builtin_amdgcn_readlane(ids, lt - lw);
      tok = lp.key0 + lt * kShTile + 16 * w;
      kvh = lp.kvh;
      hi = lp.hi;
      ++lpos;
      ++lt;
      if (lpos < last) {
        if (lt == lp.t1) {
          lp = locate(lpos);
          lt = lw = lp.t0;
          ids = load_ids(lp, lw);
        } else if (lt - lw == kShIds) {
          lw = lt;
          ids = load_ids(lp, lw);
        }
      }
    }
    const bool in = phys >= 0 && phys < p.num_blocks;
    const int slot = tok - page_of(tok) * p.bs;
    const int64_t off = in ? static_cast<int64_t>(phys) * p.blk_stride +
                                 static_cast<int64_t>(slot) * p.slot_stride +
                                 static_cast<int64_t>(kvh) * p.head_stride
                           : 0;
    const int nbytes = in ? static_cast<int>((min(16, hi - tok) - 1) * row_bytes + D * EB) : 0;
    const __amdgpu_buffer_rsrc_t rk = tile_rsrc(kbase + off, nbytes);
    const __amdgpu_buffer_rsrc_t rv = tile_rsrc(vbase + off, nbytes);
    if constexpr (WIDEN) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        k_held[set][j] = buffer_load16<2>(rk, dvo[j]);
        v_held[set][j] = buffer_load16<2>(rv, dvo[j]);
      }
      live_held[set] = in ? 1 : 0;
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j) lds_copy16(rk, sk + (16 * w + RPI * j) * D, dvo[j]);
#pragma unroll
      for (int j = 0; j < NI; ++j) lds_copy16(rv, sv + (16 * w + RPI * j) * D, dvo[j]);
      if (lane == 0) s_live[buf][w] = in ? 1 : 0;
    }
  };
  // fp8: the held set's rows, widened, into the slot.
  auto land = [&](uint16_t* sk, uint16_t* sv, int buf, auto set_c) __attribute__((always_inline)) {
    constexpr int set = decltype(set_c)::value;
    if constexpr (WIDEN) {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int lr = RPI * j + lane / CPR;
        const int c = 2 * (lane % CPR);
        typedef typename KV::raw_t raw_t;
        const uint4 a = k_held[set][j], b = v_held[set][j];
        uint16_t* const rk = sk + (16 * w + lr) * D;
        uint16_t* const rv = sv + (16 * w + lr) * D;
        *reinterpret_cast<uint4*>(rk + 8 * (c ^ pf_swz<D>(lr))) = KV::operand(raw_t{a.x, a.y});
        *reinterpret_cast<uint4*>(rk + 8 * ((c + 1) ^ pf_swz<D>(lr))) = KV::operand(raw_t{a.z, a.w});
        *reinterpret_cast<uint4*>(rv + 8 * (c ^ pf_swz<D>(lr))) = KV::operand(raw_t{b.x, b.y});
        *reinterpret_cast<uint4*>(rv + 8 * ((c + 1) ^ pf_swz<D>(lr))) = KV::operand(raw_t{b.z, b.w});
      }
      if (lane == 0) s_live[buf][w] = live_held[set];
    }
  };

  // ---- a piece's query rows ----
  uint4 qb[JD];       // the B operand Q^T: row n, dims 8 (4 j + g) ..
  int hi_n = 0;       // the lane's row sees keys below hi_n
  int wave_all = 0;   // every row of the wave sees keys below wave_all,
  int wave_any = 0;   // none sees one at or past wave_any
  int64_t orow = -1;  // the row's place in the output, -1: none
  int RW = 1, rw = 0, ks = 0, KS = 1;  // the wave takes rows 16 rw .., every KS-th 32-key block
  float m_run, l_run;
  mf_f32x4 acc[ND];
  auto begin = [&](const Piece& c) __attribute__((always_inline)) {
    RW = c.nrows > 64 ? 8 : (c.nrows > 32 ? 4 : (c.nrows > 16 ? 2 : 1));
    rw = w & (RW - 1);
    KS = kShWaves / RW;
    ks = w / RW;
    const int r = 16 * rw + n;
    hi_n = 0;
    orow = -1;
    if (r < c.nrows) {
      const int row = c.row0 + r;
      const int member = row / RPS;
      const int rest = row - member * RPS;
      const int i = rest / p.G;
      const int b = c.b0 + member;
      orow = (static_cast<int64_t>(b) * p.q_len + i) * p.H + c.kvh * p.G + (rest - i * p.G);
      hi_n = min(c.hi, s_len[b] - p.q_len + i + 1);
    }
    const T* const q = static_cast<const T*>(p.q) + (orow < 0 ? 0 : orow) * D;
#pragma unroll
    for (int j = 0; j < JD; ++j) qb[j] = *reinterpret_cast<const uint4*>(q + 8 * (4 * j + g));
    int lo = orow < 0 ? INT_MAX : hi_n, hi = hi_n;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      lo = min(lo, __shfl_xor(lo, o, kWave));
      hi = max(hi, __shfl_xor(hi, o, kWave));
    }
    wave_all = uni(lo);
    wave_any = uni(hi);
    m_run = -INFINITY;
    l_run = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t) acc[t] = mf_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  };

  // ---- one tile: the wave's 32-key blocks ks, ks + KS, .. ----
  const uint32_t kx = static_cast<uint32_t>(n * 2 * D);
  const int vtok = 4 * g + (n >> 2);  // the token a lane names in a transposed read, and its dims
  auto tile = [&](const uint16_t* sk, const uint16_t* sv, int buf, const Piece& c, int t)
                  __attribute__((always_inline)) {
    const int key_t = c.key0 + t * kShTile;
    for (int kb = ks; kb < kShTile / 32; kb += KS) {
      const int key = key_t + 32 * kb;
      if (key >= wave_any) break;
      const int live = uni(s_live[buf][2 * kb]) & 1, live2 = uni(s_live[buf][2 * kb + 1]) & 1;
      mf_f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = mf_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const char* const base = reinterpret_cast<const char*>(sk) + (32 * kb + 16 * h) * 2 * D + kx;
#pragma unroll
        for (int j = 0; j < JD; ++j)
          s[h] = Mfma16<T>::mac(
              *reinterpret_cast<const uint4*>(base + 16 * ((4 * j + g) ^ pf_swz<D>(n))), qb[j], s[h]);
      }
      float sc[8];
      const bool full = key + 32 <= wave_all && live && live2;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sc[4 * h + r] = s[h][r] * p.scale_log2;
          if (!full) {
            const bool ok = (h ? live2 : live) && key + 16 * h + 4 * g + r < hi_n;
            sc[4 * h + r] = ok ? sc[4 * h + r] : -INFINITY;
          }
        }
      float mt = sc[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mt = fmaxf(mt, sc[e]);
      const float m_new = fmaxf(m_run, rows4_max(mt));
      const bool some = m_new != -INFINITY;
      const float alpha = some ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.0f;
      const float m_use = some ? m_new : 0.0f;  // (masked scores weigh 2^-inf = 0, NaN stays NaN)
      float pr[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) pr[e] = __builtin_amdgcn_exp2f(sc[e] - m_use);
      // The weights are rounded to the query type for the matrix cores (half a step of it, at
      // most 1); l sums the rounded ones, so that the weights used still sum to one.
      const uint4 pb = make_uint4(Pack2<T>::pack(pr[0], pr[1]), Pack2<T>::pack(pr[2], pr[3]),
                                  Pack2<T>::pack(pr[4], pr[5]), Pack2<T>::pack(pr[6], pr[7]));
      const uint32_t one2 = Pack2<T>::pack(1.0f, 1.0f);
      l_run = fmaf(l_run, alpha,
                   Dot2<T>::dot(pb.w, one2, Dot2<T>::dot(pb.z, one2, Dot2<T>::dot(pb.y, one2,
                   Dot2<T>::dot(pb.x, one2, 0.0f)))));
      m_run = m_new;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int u = 0; u < ND; ++u) acc[u] *= alpha;
      }
      const char* const vb = reinterpret_cast<const char*>(sv) + (32 * kb + vtok) * 2 * D + 8 * (n & 1);
#pragma unroll
      for (int u = 0; u < ND; ++u) {
        const int ch = 2 * u + ((n & 3) >> 1);  // the 16-byte chunk of dims 16 u + 4 (n & 3)
        const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s4*)(vb + 16 * (ch ^ pf_swz<D>(vtok)))));
        const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s4*)(vb + 16 * 2 * D + 16 * (ch ^ pf_swz<D>(vtok)))));
        acc[u] = Mfma16<T>::mac(make_uint4(a.x, a.y, b.x, b.y), pb, acc[u]);
      }
    }
  };

  // ---- a piece's end: its key-splitting waves are joined through the tile's slot (read for the
  // last time before the barrier that precedes this), and the partials stored ----
  constexpr int kSlotF4 = ND * kWave;  // float4 a wave's accumulators take
  static_assert(4 * kSlotF4 * 16 == sizeof(s_k0), "four waves' accumulators fill a K slot");
  auto finish = [&](uint16_t* sk, uint16_t* sv, const Piece& c) __attribute__((always_inline)) {
    l_run = rows4_sum(l_run);
    auto slot_of = [&](int i) {
      return (i < 4 ? reinterpret_cast<float4*>(sk) + i * kSlotF4
                    : reinterpret_cast<float4*>(sv) + (i - 4) * kSlotF4) + lane;
    };
    const int KA = min(KS, kShTile / 32);  // waves of a row block that took keys
    if (KA > 1) {
      if (ks > 0 && ks < KA) {
        float4* const d = slot_of((ks - 1) * RW + rw);
#pragma unroll
        for (int u = 0; u < ND; ++u)
          d[u * kWave] = make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
        if (g == 0) s_ml[w][n] = make_float2(m_run, l_run);
      }
      __syncthreads();
      if (ks == 0) {
        for (int k = 1; k < KA; ++k) {
          const float2 ml = s_ml[k * RW + rw][n];
          const float M = fmaxf(m_run, ml.x);
          const bool some = M != -INFINITY;
          const float a0 = some ? __builtin_amdgcn_exp2f(m_run - M) : 1.0f;
          const float a1 = some ? __builtin_amdgcn_exp2f(ml.x - M) : 0.0f;
          const float4* const d = slot_of((k - 1) * RW + rw);
#pragma unroll
          for (int u = 0; u < ND; ++u) {
            const float4 o = d[u * kWave];
            acc[u][0] = fmaf(o.x, a1, acc[u][0] * a0);
            acc[u][1] = fmaf(o.y, a1, acc[u][1] * a0);
            acc[u][2] = fmaf(o.z, a1, acc[u][2] * a0);
            acc[u][3] = fmaf(o.w, a1, acc[u][3] * a0);
          }
          l_run = fmaf(ml.y, a1, l_run * a0);
          m_run = M;
        }
      }
    }
    if (ks == 0 && orow >= 0) {
      const int64_t slot = c.t0 == 0 ? c.kind * p.rows + orow
                                     : 2 * p.rows + static_cast<int64_t>(share) * kShRows + 16 * rw + n;
      if (g == 0) *reinterpret_cast<float2*>(p.ml + 2 * slot) = make_float2(m_run, l_run);
      float* const a = p.acc + slot * D + 4 * g;
#pragma unroll
      for (int u = 0; u < ND; ++u)
        *reinterpret_cast<float4*>(a + 16 * u) = make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
    }
    if (KA > 1) __syncthreads();  // the slot is free again
  };

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  Piece cp = lp;
  int cpos = first, ct = cp.t0;
  request(s_k0, s_v0, 0, I0{});
  if constexpr (WIDEN) {
    request(s_k1, s_v1, 1, I1{});
    land(s_k0, s_v0, 0, I0{});
    request(s_k0, s_v0, 0, I0{});
    land(s_k1, s_v1, 1, I1{});
    request(s_k1, s_v1, 1, I1{});
  } else {
    request(s_k1, s_v1, 1, I1{});
  }
  begin(cp);
  // Tile cpos sits in slot `buf`; after it the slot takes tile cpos + 2 (fp8: which set `buf`
  // holds, while the set takes tile cpos + 4).
  auto step = [&](uint16_t* sk, uint16_t* sv, int buf, auto set_c) __attribute__((always_inline)) {
    // tile cpos has landed: everything but the last tile requested
    if constexpr (!WIDEN) __builtin_amdgcn_s_waitcnt(sh_wait_vm(2 * NI));
    __syncthreads();
    tile(sk, sv, buf, cp, ct);
    __syncthreads();  // the slot has been read
    ++cpos;
    ++ct;
    if (ct == cp.t1) {
      finish(sk, sv, cp);
      if (cpos < last) {
        cp = locate(cpos);
        ct = cp.t0;
        begin(cp);
      }
    }
    land(sk, sv, buf, set_c);
    request(sk, sv, buf, set_c);
  };
  while (true) {
    step(s_k0, s_v0, 0, I0{});
    if (cpos >= last) break;
    step(s_k1, s_v1, 1, I1{});
    if (cpos >= last) break;
  }
  // (copies of tiles past the share read nothing; they land before the workgroup's LDS is given
  // to another)
  __builtin_amdgcn_s_waitcnt(sh_wait_vm(0));
}

// Joins a row's pieces: one wave a query row, D / 64 dims a lane. Its pieces: for the group's
// segment (if the row has one) and for its own, the unit's first piece, then those of the shares
// that the unit runs on into.
constexpr int kShMergeThreads = 256;
constexpr int kShMergeWaves = kShMergeThreads / kWave;
template <typename T, int D>
__global__ __launch_bounds__(kShMergeThreads) void shared_merge_kernel(const SharedParams p) {
  constexpr int DPL = D / 64;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kShMergeWaves +
                      __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  if (row >= p.rows) return;
  const int B = p.batch, NG = p.groups, NS = NG + B;
  const int* const cum = p.plan + kShPlanCum;
  const int bi = static_cast<int>(row / p.H);
  const int h = static_cast<int>(row - static_cast<int64_t>(bi) * p.H);
  const int b = bi / p.q_len, i = bi - b * p.q_len;
  const int kvh = h / p.G, gq = h - kvh * p.G;
  const int RPS = p.q_len * p.G;
  const int per = p.plan[0];
  const int grp = cum[NS + 1 + b];
  float M = -INFINITY, L = 0.0f;
  float o[DPL];
#pragma unroll
  for (int d = 0; d < DPL; ++d) o[d] = 0.0f;
  auto take = [&](int64_t slot) __attribute__((always_inline)) {
    const float2 ml = *reinterpret_cast<const float2*>(p.ml + 2 * slot);
    float a[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) a[d] = p.acc[slot * D + DPL * lane + d];
    const float Mn = fmaxf(M, ml.x);
    const bool some = Mn != -INFINITY;
    const float w0 = some ? __builtin_amdgcn_exp2f(M - Mn) : 1.0f;
    const float w1 = some ? __builtin_amdgcn_exp2f(ml.x - Mn) : 0.0f;
    L = fmaf(ml.y, w1, L * w0);
#pragma unroll
    for (int d = 0; d < DPL; ++d) o[d] = fmaf(a[d], w1, o[d] * w0);
    M = Mn;
  };
  for (int kind = 0; kind < 2; ++kind) {
    if (kind == 0 && grp < 0) continue;
    const int seg = kind == 0 ? grp : NG + b;
    const int c0 = cum[seg], c1 = cum[seg + 1];
    if (c1 <= c0) continue;
    int r = i * p.G + gq, members = 1;
    if (kind == 0) {
      const int* const g0 = cum + NS + 1 + B;
      r += (b - g0[grp]) * RPS;
      members = g0[grp + 1] - g0[grp];
    }
    const int rtiles = ceil_div(members * RPS, kShRows);
    const int tiles = (c1 - c0) / (rtiles * p.KVH);
    const int t0 = c0 + (kvh * rtiles + r / kShRows) * tiles;
    const int s0 = t0 / per, s1 = (t0 + tiles - 1) / per;
    take(kind * p.rows + row);
    for (int s = s0 + 1; s <= s1 && s < p.shares; ++s)
      take(2 * p.rows + static_cast<int64_t>(s) * kShRows + r % kShRows);
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
  hipLaunchKernelGGL((shared_merge_kernel<T, D>), dim3(static_cast<unsigned>(blocks)),
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
