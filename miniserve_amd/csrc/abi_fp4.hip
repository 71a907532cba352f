// C ABI of the 4-bit paged cache (declared in include/msattn.h): argument checks and launches.
// No exception crosses this boundary.
#include <cmath>
#include <cstdint>

#include <algorithm>

#include "fp4_attn.h"
#include "msattn.h"

namespace {

using namespace msattn;

bool on(const void* p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
bool float_type(int t) { return t == MSATTN_F32 || t == MSATTN_F16 || t == MSATTN_BF16; }
int type_bytes(int t) { return t == MSATTN_F32 ? 4 : 2; }
bool dim_ok(int D) { return D > 0 && D % kFp4Block == 0 && D <= kFp4MaxDim; }

// The caches lie on 16 bytes, and so do their pages and heads.
bool cache_ok(const void* k, const void* v, int64_t blk, int64_t head, int KVH, int D, int bs,
              int num_blocks, int W) {
  return k && v && on(k, 16) && on(v, 16) && blk >= 0 && head >= 0 && blk % 16 == 0 &&
         head % 16 == 0 && KVH > 0 && dim_ok(D) && bs > 0 && bs % kFp4Tile == 0 && num_blocks > 0 &&
         W > 0;
}

// A launch has fewer than 2^32 threads.
bool grid_ok(int64_t workgroups, int threads) { return workgroups * threads < (int64_t(1) << 32); }

int status_of(hipError_t e) { return e == hipSuccess ? MSATTN_OK : MSATTN_ERR_HIP; }

// Write or read: the parameters that both have.
int cache_params(Fp4CacheParams* p, const void* k, const void* v, const int64_t* ks,
                 const int64_t* vs, void* k_cache, void* v_cache, int64_t blk, int64_t head,
                 const int32_t* table, const int32_t* starts, int batch, int tokens, int KVH, int D,
                 int bs, int num_blocks, int W, int dtype) {
  if (!k || !v || !table || !starts || batch <= 0 || tokens < 0 || !float_type(dtype) ||
      !cache_ok(k_cache, v_cache, blk, head, KVH, D, bs, num_blocks, W))
    return MSATTN_ERR_INVALID_ARG;
  const int eb = type_bytes(dtype);
  if (!on(k, eb) || !on(v, eb) || !on(table, 4) || !on(starts, 4)) return MSATTN_ERR_INVALID_ARG;
  // tokens positions from anywhere in a tile, a wave for each tile they may touch
  p->tiles = static_cast<int>((static_cast<int64_t>(tokens) + 2 * (kFp4Tile - 1)) / kFp4Tile);
  p->items = static_cast<int64_t>(batch) * p->tiles;
  if (p->items >= (int64_t(1) << 31) || !grid_ok(p->items *= KVH, 64) ||
      !grid_ok(fp4_cache_workgroups(p->items), kFp4CacheThreads))
    return MSATTN_ERR_UNSUPPORTED;
  p->k_cache = static_cast<uint8_t*>(k_cache);
  p->v_cache = static_cast<uint8_t*>(v_cache);
  p->k = const_cast<void*>(k);
  p->v = const_cast<void*>(v);
  p->table = table;
  p->starts = starts;
  p->blk_stride = blk;
  p->head_stride = head;
  p->vec = on(k, 16) && on(v, 16);
  for (int i = 0; i < 3; ++i) {
    p->k_st[i] = ks[i];
    p->v_st[i] = vs[i];
    if (ks[i] * eb % 16 != 0 || vs[i] * eb % 16 != 0) p->vec = 0;
  }
  p->batch = batch;
  p->tokens = tokens;
  p->KVH = KVH;
  p->D = D;
  p->bs = bs;
  p->num_blocks = num_blocks;
  p->W = W;
  p->by_tiles = fp4_div(static_cast<uint32_t>(p->tiles > 0 ? p->tiles : 1));
  p->by_heads = fp4_div(static_cast<uint32_t>(KVH));
  p->by_bs = fp4_div(static_cast<uint32_t>(bs));
  return MSATTN_OK;
}

bool geometry_ok(int batch, int q_len, int H, int KVH, int D, int max_ctx) {
  return batch > 0 && q_len > 0 && H > 0 && KVH > 0 && H % KVH == 0 && dim_ok(D) && max_ctx >= 0;
}

// How a call is cut: the way, blocks of 16 query rows a wave, waves of a unit, shares or parts.
struct Plan {
  int way, ct, wk, rblocks, slot_rows, shares, parts, xcd_units;
  size_t ml_off, acc_off, total;
};

int64_t ceil_div64(int64_t a, int64_t b) { return (a + b - 1) / b; }

size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// A wave's time for a group with 64 query rows over that with 32: less than twice, since the keys and
// values are widened once. 512 queries of H28/KVH4/D128 behind 4096 keys, 2 rows: 103 us against 111;
// 1024 queries of H32/KVH8/D128 by themselves, 4 rows, where half as many units fill the CUs less
// evenly: 99 against 90, and this factor chooses the latter.
constexpr double kRound64 = 1.8;

// And with 16. 32 rows of 4 drafts of H28/KVH4/D128 under a window of 2048, 128 units of 28 rows: 24.1
// us, as 256 of 16 18.6; the chunk above 147.
constexpr double kRound16 = 0.65;

// Contexts go up to this: a position plus a query's offset or a window fits 31 bits.
constexpr int kMaxContext = 1 << 30;

// Workspace does not depend on causal and window.
bool plan_of(int batch, int q_len, int H, int KVH, int D, int max_ctx, int causal,
             int window, int q_dtype, Plan* p) {
  const int G = H / KVH;
  const int64_t rows = static_cast<int64_t>(q_len) * G;
  const int DP = D <= 64 ? 64 : (D <= 128 ? 128 : 256);
  const int parts = q_dtype == MSATTN_BF16 ? 1 : (q_dtype == MSATTN_F16 ? 2 : 3);
  const int list_ct = fp4_list_ct(parts, DP), max_ct = fp4_max_ct(parts, DP);
  p->ct = rows <= 16 ? 1 : list_ct;
  const int per = 16 * p->ct;
  const int64_t rblocks = (rows + per - 1) / per;
  const int64_t units = batch * rblocks * KVH;
  if (rows >= (int64_t(1) << 30) || units >= (int64_t(1) << 30) || max_ctx > kMaxContext) return false;
  p->rblocks = static_cast<int>(rblocks);
  p->slot_rows = static_cast<int>(std::min<int64_t>(per, rows));
  const int64_t want = kFp4Shares;  // workgroups: one a CU
  int64_t groups = max_ctx / kFp4Group + 1;  // of a unit, at most
  const bool split = batch * rblocks <= kFp4MaxEntries && units * (groups + kFp4Head) < (int64_t(1) << 30);
  p->way = split ? kFp4List : kFp4Dealt;
  p->parts = 1;
  p->shares = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, units * (groups + kFp4Head))));
  const size_t slots = split ? 2 * static_cast<size_t>(p->shares) * p->slot_rows : 0;
  p->ml_off = up256((kHdrTickets + kMaxTickets) * sizeof(int));
  p->acc_off = p->ml_off + up256(slots * 2 * sizeof(float));
  p->total = p->acc_off + up256(slots * D * sizeof(float));
  if (window > 0)
    groups = std::min<int64_t>(groups, (static_cast<int64_t>(window) + per / G + 1) / kFp4Group + 2);
  // Without a list, partials and joins: whole units, wk waves each. What each way costs, in a wave's
  // groups (about 1.3 us at 32 rows, two waves a SIMD): a unit's start and end are about 3 of them,
  // and about 10 each with a list (its plan, partials and joins, in which all waves of a workgroup
  // meet). Several rounds of the CUs even out; the last unit to start does not. Measured: 896 units of
  // 32 rows and 144 groups, wk = 1, 2, 4, 8 and the list, 210, 111, 113, 124, 161 us; of 65 groups 101,
  // 58, 59, 70, 105; 4096 of 32, causal, 105, 90, 114, 160, 301. Units of few rows take all waves of a
  // workgroup.
  const double mean = groups - (causal && window == 0 ? 0.5 * std::min(q_len, max_ctx) / kFp4Group : 0.0);
  const double listed = static_cast<double>(units) / want;  // units a CU
  double best = 1e300;
  if (split)
    best = (rows > 16 && list_ct == 1 ? kRound16 : 1.0) * listed * mean / kFp4Waves + 10 * (listed + 1);
  p->wk = kFp4Waves;
  auto consider = [&](int ct, int wk, double round) {  // round: of a group of 16 ct rows
    const int64_t blocks = (rows + 16 * ct - 1) / (16 * ct);
    const double load = static_cast<double>(batch * blocks * KVH) / want;
    const double longest = ceil(static_cast<double>(groups) / wk) + 3, rounds = load * wk / kFp4Waves;
    const double cost = round * (rounds <= 1 ? longest : rounds * (mean / wk + 3) + 0.5 * longest);
    if (cost > best) return;
    best = cost;
    p->ct = ct;
    p->wk = wk;
    p->way = kFp4Dealt;
    p->rblocks = static_cast<int>(blocks);
  };
  if (rows <= 16) {
    // Where a CU gets several units of few rows, in us: dealt, each round of them starts anew (about 3.7
    // on top of 5), and a list shares their groups evenly (10, 5 a unit and CU). Dealt units take longer
    // for their groups where these stream at the memory's rate, bf16 above 64 dims, than where the
    // waves' own work bounds them. List / dealt: H32/KVH8/D128, 64 rows of 640 keys 19.5 / 17.5, of 1300
    // 33.5 / 25.8, of 1024 to 8192 49.5 / 59.6; 100 rows of 1000 39.6 / 36.4, of 2500 62.7 / 65.4; in
    // fp32 64 of 2500 55.0 / 44.0; H12/KVH12/D64, 64 of 2500 51.8 / 30.1, 100 in fp32 82.1 / 71.8. (64 of
    // 5000 there, which these figures leave to a list: 77.7 / 50.1.)
    const double slower = parts > 1 || D <= 64 ? 0.2 : 0.45;  // us a wave's group
    const bool few = slower * listed * groups / kFp4Waves < 5 + 1.3 * listed;
    if (split && listed > 1) best = few ? 1e300 : 0;
    consider(1, kFp4Waves, 1.0);
  } else {
    for (int wk = kFp4Waves; wk >= 1; wk /= 2) consider(1, wk, kRound16);
    for (int wk = kFp4Waves; max_ct >= 2 && wk >= 1; wk /= 2) consider(2, wk, 1.0);
    if (max_ct == 4 && rows > 32)
      for (int wk = 4; wk >= 1; wk /= 2) consider(4, wk, kRound64);
  }
  // Few units: each cut into as many parts as there are CUs for it, a workgroup a part, joined like
  // shares but without a list's plan. Start, partials and join cost 7 groups, 5 of the longer ones above
  // 128 dims. List / parts: 16 rows of 1024 to 4096 keys of H28/KVH4/D128 in fp16 20.7 / 16.1 us, 16 of
  // 16384 of H32/KVH8/D128 58.6 / 51.8, 32 of 1024 to 8192 of H8/KVH1/D256 in fp32 42.1 / 31.5. Dealt /
  // parts: 4 rows of H32/KVH8/D128 up to 600 keys 9.0 / 11.1, 1000 10.8 / 11.3, 1400 12.3 / 11.4, 2000
  // 14.5 / 12.0; 16 of H8/KVH1/D256 up to 600 13.9 / 13.3, 2000 22.8 / 14.6.
  const int64_t most = std::min<int64_t>(want / units, (groups + kFp4Waves - 1) / kFp4Waves);
  if (split && most > 1) {
    const double cost = (rows > 16 && list_ct == 1 ? kRound16 : 1.0) *
                            ceil(static_cast<double>(groups) / (most * kFp4Waves)) +
                        (D > 128 ? 5 : 7);
    if (cost < best) {
      p->way = kFp4Parts;
      p->ct = rows <= 16 ? 1 : list_ct;
      p->wk = kFp4Waves;
      p->rblocks = static_cast<int>(rblocks);
      p->parts = static_cast<int>(most);
    }
  }
  const int64_t dealt = static_cast<int64_t>(batch) * p->rblocks * KVH * p->parts;  // units, or parts of them
  p->xcd_units = static_cast<int>(ceil_div64(ceil_div64(dealt * p->wk, kFp4Waves), 8));
  return true;
}

bool launch_ok(const Plan& p) {
  return p.way == kFp4List || grid_ok(8 * static_cast<int64_t>(p.xcd_units), kFp4Threads);
}

}  // namespace

extern "C" {

int msattn_write_kv_fp4(const void* k, int64_t k_batch_stride, int64_t k_token_stride,
                        int64_t k_head_stride, const void* v, int64_t v_batch_stride,
                        int64_t v_token_stride, int64_t v_head_stride, void* k_cache,
                        void* v_cache, int64_t cache_block_stride, int64_t cache_head_stride,
                        const int32_t* block_table, const int32_t* starts, int batch, int tokens,
                        int num_kv_heads, int head_dim, int block_size, int num_blocks,
                        int table_width, int src_dtype, void* stream) {
  const int64_t ks[3] = {k_batch_stride, k_token_stride, k_head_stride};
  const int64_t vs[3] = {v_batch_stride, v_token_stride, v_head_stride};
  for (int i = 0; i < 3; ++i)
    if (ks[i] < 0 || vs[i] < 0) return MSATTN_ERR_INVALID_ARG;
  Fp4CacheParams p{};
  const int rc = cache_params(&p, k, v, ks, vs, k_cache, v_cache, cache_block_stride,
                              cache_head_stride, block_table, starts, batch, tokens, num_kv_heads,
                              head_dim, block_size, num_blocks, table_width, src_dtype);
  if (rc != MSATTN_OK || tokens == 0) return rc;
  // The bytes that k, v and the caches span.
  const int eb = type_bytes(src_dtype);
  const int64_t cache_span = (num_blocks - 1) * cache_block_stride +
                             (num_kv_heads - 1) * cache_head_stride +
                             static_cast<int64_t>(block_size / kFp4Tile) * fp4_tile_bytes(head_dim);
  const struct { const void* at; const int64_t* st; } in[2] = {{k, ks}, {v, vs}};
  for (const auto& x : in) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(x.at);
    const uintptr_t hi = lo + static_cast<uintptr_t>(((batch - 1) * x.st[0] + (tokens - 1) * x.st[1] +
                                                      (num_kv_heads - 1) * x.st[2] + head_dim) * eb);
    for (const void* c : {static_cast<const void*>(k_cache), static_cast<const void*>(v_cache)}) {
      const uintptr_t clo = reinterpret_cast<uintptr_t>(c);
      if (lo < clo + static_cast<uintptr_t>(cache_span) && clo < hi) return MSATTN_ERR_OVERLAP;
    }
  }
  return status_of(launch_write_fp4(p, src_dtype, static_cast<hipStream_t>(stream)));
}

int msattn_read_kv_fp4(const void* k_cache, const void* v_cache, int64_t cache_block_stride,
                       int64_t cache_head_stride, const int32_t* block_table,
                       const int32_t* starts, void* k, void* v, int batch, int tokens,
                       int num_kv_heads, int head_dim, int block_size, int num_blocks,
                       int table_width, int dst_dtype, void* stream) {
  Fp4CacheParams p{};
  const int64_t st[3] = {static_cast<int64_t>(tokens) * num_kv_heads * head_dim,
                         static_cast<int64_t>(num_kv_heads) * head_dim, head_dim};
  const int rc = cache_params(&p, k, v, st, st, const_cast<void*>(k_cache),
                              const_cast<void*>(v_cache), cache_block_stride, cache_head_stride,
                              block_table, starts, batch, tokens, num_kv_heads, head_dim,
                              block_size, num_blocks, table_width, dst_dtype);
  if (rc != MSATTN_OK || tokens == 0) return rc;
  return status_of(launch_read_fp4(p, dst_dtype, static_cast<hipStream_t>(stream)));
}

size_t msattn_fp4_workspace_bytes(int batch, int q_len, int num_heads, int num_kv_heads,
                                  int head_dim, int max_context, int q_dtype) {
  Plan plan;
  if (!geometry_ok(batch, q_len, num_heads, num_kv_heads, head_dim, max_context) ||
      !float_type(q_dtype) ||
      !plan_of(batch, q_len, num_heads, num_kv_heads, head_dim, max_context, 1, 0, q_dtype, &plan))
    return 0;
  return plan.total;
}

int msattn_fp4_plan(int batch, int q_len, int num_heads, int num_kv_heads, int head_dim,
                    int max_context, int causal, int window, int q_dtype, int* plan) {
  Plan p;
  if (!plan || window < 0 || !float_type(q_dtype) ||
      !geometry_ok(batch, q_len, num_heads, num_kv_heads, head_dim, max_context))
    return MSATTN_ERR_INVALID_ARG;
  if (!plan_of(batch, q_len, num_heads, num_kv_heads, head_dim, max_context, causal, window, q_dtype, &p) ||
      !launch_ok(p))
    return MSATTN_ERR_UNSUPPORTED;
  plan[0] = p.way;
  plan[1] = p.ct;
  plan[2] = p.wk;
  plan[3] = p.parts;
  return MSATTN_OK;
}

int msattn_paged_attention_fp4(const void* query, int64_t q_batch_stride,
                               int64_t q_token_stride, int64_t q_head_stride,
                               const void* k_cache, const void* v_cache,
                               int64_t cache_block_stride, int64_t cache_head_stride,
                               const int32_t* block_table,
                               const int32_t* context_lens, void* out, void* workspace,
                               size_t workspace_bytes, int batch, int q_len, int num_heads,
                               int num_kv_heads, int head_dim, int block_size, int num_blocks,
                               int table_width, int max_context, int causal, int window,
                               float scale, int q_dtype, void* stream) {
  if (!query || !block_table || !context_lens || !out || !workspace ||
      !float_type(q_dtype) || window < 0 || std::isnan(scale) ||
      !geometry_ok(batch, q_len, num_heads, num_kv_heads, head_dim, max_context) ||
      !cache_ok(k_cache, v_cache, cache_block_stride, cache_head_stride, num_kv_heads, head_dim,
                block_size, num_blocks, table_width))
    return MSATTN_ERR_INVALID_ARG;
  const int eb = type_bytes(q_dtype);
  if (!on(query, 16) || !on(out, 16) || !on(workspace, 256) || !on(block_table, 4) ||
      !on(context_lens, 4))
    return MSATTN_ERR_INVALID_ARG;
  const int64_t q_strides[3] = {q_batch_stride, q_token_stride, q_head_stride};
  for (int64_t x : q_strides)
    if (x < 0 || x * eb % 16 != 0) return MSATTN_ERR_INVALID_ARG;
  Plan plan;
  if (!plan_of(batch, q_len, num_heads, num_kv_heads, head_dim, max_context, causal, window, q_dtype, &plan) ||
      !launch_ok(plan))
    return MSATTN_ERR_UNSUPPORTED;
  if (workspace_bytes < plan.total) return MSATTN_ERR_WORKSPACE;
  char* const ws = static_cast<char*>(workspace);
  Fp4Params p{};
  p.q = query;
  p.k = static_cast<const uint8_t*>(k_cache);
  p.v = static_cast<const uint8_t*>(v_cache);
  p.table = block_table;
  p.lens = context_lens;
  p.out = out;
  p.blk_stride = cache_block_stride;
  p.head_stride = cache_head_stride;
  for (int i = 0; i < 3; ++i) p.q_st[i] = q_strides[i];
  p.batch = batch;
  p.q_len = q_len;
  p.H = num_heads;
  p.KVH = num_kv_heads;
  p.G = num_heads / num_kv_heads;
  p.D = head_dim;
  p.bs = block_size;
  p.num_blocks = num_blocks;
  p.W = table_width;
  // (no key past the table)
  p.max_ctx = static_cast<int>(std::min<int64_t>(
      max_context, static_cast<int64_t>(table_width) * block_size));
  p.causal = causal != 0;
  p.window = window < p.max_ctx ? window : 0;  // (one as long as any context hides nothing)
  p.scale_log2 = scale * kLog2e;
  p.rows_per_kvh = q_len * p.G;
  p.rblocks = plan.rblocks;
  p.slot_rows = plan.slot_rows;
  p.parts = plan.parts;
  p.shares = plan.shares;
  p.xcd_units = plan.xcd_units;
  p.by_tiles = fp4_div(static_cast<uint32_t>(block_size / kFp4Tile));
  p.by_g = fp4_div(static_cast<uint32_t>(p.G));
  p.by_rb = fp4_div(static_cast<uint32_t>(plan.rblocks));
  p.by_parts = fp4_div(static_cast<uint32_t>(plan.parts));
  p.by_kvh = fp4_div(static_cast<uint32_t>(num_kv_heads));
  p.by_per = fp4_div(static_cast<uint32_t>(head_dim / 4));
  p.tickets = reinterpret_cast<int*>(ws) + kHdrTickets;
  p.ml = reinterpret_cast<float*>(ws + plan.ml_off);
  p.acc = reinterpret_cast<float*>(ws + plan.acc_off);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&](auto t) {
    typedef decltype(t) T;
    if (head_dim <= 64) return launch_fp4_attn<T, 64>(p, plan.way, plan.ct, plan.wk, st);
    if (head_dim <= 128) return launch_fp4_attn<T, 128>(p, plan.way, plan.ct, plan.wk, st);
    return launch_fp4_attn<T, 256>(p, plan.way, plan.ct, plan.wk, st);
  };
  switch (q_dtype) {
    case MSATTN_F32: return status_of(launch(float{}));
    case MSATTN_F16: return status_of(launch(_Float16{}));
    default: return status_of(launch(bf16_t{}));
  }
}

}  // extern "C"
