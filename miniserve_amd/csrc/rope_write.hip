// The rotation of a step's queries and keys, and the scatter of the rotated keys and of the
// values into the paged cache, in one launch (msattn_write_kv_rope).
//
// Of a token at position p, for a row x of head_dim D and rotary size R <= D (even):
//   y[d] = x[d] cos[p][d] - x[d + R/2] sin[p][d]   for d < R/2,
//   y[d] = x[d] cos[p][d] + x[d - R/2] sin[p][d]   for R/2 <= d < R,
//   y[d] = x[d]                                    for R <= d < D
// (miniserve/attention.py:41-62 with fp32 tables; every product and the sum rounded on its own
// in fp32, as the decode kernels rotate a query). Query rows are rounded once to the query type;
// key rows once to the cache type, straight from fp32 (a bf16 key bound for an fp8 cache is not
// rounded to bf16 first); value rows are converted as write_kv converts them. The scatter is
// write_kv's (miniserve/attention.py:111-133): position p of sequence b lands in page
// table[b][p / bs], slot p % bs, and nowhere where that page is a hole.
//
// Bound by memory: every input row is read once and every output row written once, 3 flops an
// element in between. A wave takes one token (or a slice of its rows): each lane keeps one place
// in a row, a pair of chunks R/2 apart whose 4 E table entries it loads once, and walks the
// token's query, key and value rows with it, so the fp32 tables (4 to 8 times a row's bytes)
// are read once a wave instead of once a row. Whole prompts (kRwUnroll's) pass at
// 5.2 TB/s, where a copy of 2 GiB reaches 4.9; one token of 32 sequences (14 + 2 x 2 heads of 64)
// takes 4.6 us, two chunks of 512 tokens of 28 + 2 x 4 heads of 128 7.2, most of the former the launch.
#include "kernels.h"
#include "split_kernel.h"

namespace msattn {

constexpr int kRwThreads = 256;
constexpr int kRwWaves = kRwThreads / kWave;
// Rows a lane has in flight: 2 x 2 loads of 16 bytes. (More cost resident waves: whole prompts,
// 4 x 8191 tokens of 32 + 2 x 8 heads of 128 from bf16 into an fp8 cache, 746 MB, took 144 us
// with 1 or 2 rows, 150 with 4, 163 with 6; stores past the caches 147, and fp32 ones 20 % more.)
constexpr int kRwUnroll = 2;

struct RwToken {
  int b, t;
  int64_t cache_off;  // element offset of the token's [head 0][dim 0] in the caches, -1: a hole
  int64_t table_off;  // element offset of its position's row in the rotation tables
};

__device__ __forceinline__ RwToken rw_token(const RopeWriteParams& p, int64_t token) {
  RwToken k;
  // (a batch's tokens fit 31 bits in every call but the largest: the short division)
  k.b = token < (int64_t(1) << 31) ? static_cast<int>(static_cast<uint32_t>(token) / static_cast<uint32_t>(p.tokens))
                                   : static_cast<int>(token / p.tokens);
  k.t = static_cast<int>(token - static_cast<int64_t>(k.b) * p.tokens);
  const int64_t pos = static_cast<int64_t>(p.starts[k.b]) + p.start_offset + k.t;
  int64_t rp = pos;
  if (p.position != nullptr)
    rp = p.position_per_token ? static_cast<int64_t>(p.position[token])
                              : static_cast<int64_t>(p.position[k.b]) + k.t;
  rp = rp < 0 ? 0 : (rp >= p.max_pos ? p.max_pos - 1 : rp);
  k.table_off = rp * p.R;
  k.cache_off = -1;
  const int64_t pg = pos >= 0 ? pos / p.bs : p.W;
  if (pg < p.W) {
    const int phys = p.table[static_cast<int64_t>(k.b) * p.W + pg];
    if (phys >= 0 && phys < p.num_blocks)
      k.cache_off = static_cast<int64_t>(phys) * p.blk_stride + (pos - pg * p.bs) * p.slot_stride;
  }
  return k;
}

template <int N>
struct alignas(N >= 16 ? 16 : N) RwBytes {
  unsigned char b[N];
};

// E consecutive elements of type T, loaded or stored as one vector.
template <typename T, int E>
__device__ __forceinline__ RwBytes<E * sizeof(T)> rw_load(const T* p) {
  return *reinterpret_cast<const RwBytes<E * sizeof(T)>*>(p);
}
template <typename T, int E>
__device__ __forceinline__ void rw_unpack(const RwBytes<E * sizeof(T)>& x, float (&o)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = Elt<T>::load(reinterpret_cast<const T*>(x.b) + e);
}
template <typename T, int E>
__device__ __forceinline__ void rw_store(T* p, const float (&f)[E]) {
  RwBytes<E * sizeof(T)> x;
#pragma unroll
  for (int e = 0; e < E; ++e) Elt<T>::store(reinterpret_cast<T*>(x.b) + e, f[e]);
  *reinterpret_cast<RwBytes<E * sizeof(T)>*>(p) = x;
}

// Chunks of E elements: rows, strides and tables on the vectors' alignment, R / 2 and D multiples
// of E. A row's D / E chunks make p.items pairs, one a lane: pair i < R / (2 E) is the chunks i
// and i + R / (2 E), a later one two chunks past R (or the last alone).
template <typename ST, typename KT, int E>
__global__ __launch_bounds__(kRwThreads) void rope_write_vec_kernel(const RopeWriteParams p) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * kRwWaves +
                       __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t token = unit / p.slices;
  if (token >= static_cast<int64_t>(p.batch) * p.tokens) return;
  const int slice = static_cast<int>(unit - token * p.slices);
  const RwToken k = rw_token(p, token);

  const int heads = kWave / p.items;  // rows a wave takes at a time
  const int hl = lane / p.items;
  const int item = lane - hl * p.items;
  if (hl >= heads) return;
  const int half = p.R / 2;
  const bool turns = item < half / E;
  const int c0 = turns ? item * E : p.R + 2 * (item - half / E) * E;
  const int c1 = turns ? c0 + half : c0 + E;
  const bool two = c1 < p.D;  // false: the row's odd last chunk

  float cs[2][E], sn[2][E];
  if (turns) {
    const float* ct = p.cos + k.table_off;
    const float* st = p.sin + k.table_off;
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      *reinterpret_cast<float4*>(&cs[0][e]) = *reinterpret_cast<const float4*>(ct + c0 + e);
      *reinterpret_cast<float4*>(&cs[1][e]) = *reinterpret_cast<const float4*>(ct + c1 + e);
      *reinterpret_cast<float4*>(&sn[0][e]) = *reinterpret_cast<const float4*>(st + c0 + e);
      *reinterpret_cast<float4*>(&sn[1][e]) = *reinterpret_cast<const float4*>(st + c1 + e);
    }
  }

  const ST* const qs = static_cast<const ST*>(p.q) + k.b * p.q_src[0] + k.t * p.q_src[1];
  const ST* const ks = static_cast<const ST*>(p.k) + k.b * p.k_src[0] + k.t * p.k_src[1];
  const ST* const vs = static_cast<const ST*>(p.v) + k.b * p.v_src[0] + k.t * p.v_src[1];
  ST* const qd = static_cast<ST*>(p.q_out) + k.b * p.q_dst[0] + k.t * p.q_dst[1];
  // Rows 0 .. QH - 1 are query heads, then KVH key heads, then KVH value heads (read before the
  // page is known, not written where it is a hole).
  const int QH = p.QH;
  const int rows = QH + 2 * p.KVH;
  const int step = heads * p.slices;
  for (int r0 = slice * heads + hl; r0 < rows; r0 += step * kRwUnroll) {
    RwBytes<E * sizeof(ST)> x0[kRwUnroll], x1[kRwUnroll];
#pragma unroll
    for (int u = 0; u < kRwUnroll; ++u) {
      const int r = r0 + u * step;
      if (r < rows) {
        const ST* s = r < QH           ? qs + r * p.q_src[2]
                      : r < QH + p.KVH ? ks + (r - QH) * p.k_src[2]
                                       : vs + (r - QH - p.KVH) * p.v_src[2];
        x0[u] = rw_load<ST, E>(s + c0);
        x1[u] = rw_load<ST, E>(s + (two ? c1 : c0));
      }
    }
#pragma unroll
    for (int u = 0; u < kRwUnroll; ++u) {
      const int r = r0 + u * step;
      if (r >= (k.cache_off >= 0 ? rows : QH)) continue;
      const bool value = r >= QH + p.KVH;
      if (value && std::is_same<ST, KT>::value) {  // the bits as they are
        ST* const d = static_cast<ST*>(p.v_cache) + k.cache_off + (r - QH - p.KVH) * p.head_stride;
        *reinterpret_cast<RwBytes<E * sizeof(ST)>*>(d + c0) = x0[u];
        if (two) *reinterpret_cast<RwBytes<E * sizeof(ST)>*>(d + c1) = x1[u];
        continue;
      }
      float a[E], b[E], y0[E], y1[E];
      rw_unpack<ST, E>(x0[u], a);
      rw_unpack<ST, E>(x1[u], b);
      if (turns && !value) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          y0[e] = rope_mix(a[e], -b[e], cs[0][e], sn[0][e]);
          y1[e] = rope_mix(b[e], a[e], cs[1][e], sn[1][e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          y0[e] = a[e];
          y1[e] = b[e];
        }
      }
      if (r < QH) {
        ST* const d = qd + r * p.q_dst[2];
        rw_store<ST, E>(d + c0, y0);
        if (two) rw_store<ST, E>(d + c1, y1);
      } else {
        KT* const d = (value ? static_cast<KT*>(p.v_cache) + (r - QH - p.KVH) * p.head_stride
                             : static_cast<KT*>(p.k_cache) + (r - QH) * p.head_stride) +
                      k.cache_off;
        rw_store<KT, E>(d + c0, y0);
        if (two) rw_store<KT, E>(d + c1, y1);
      }
    }
  }
}

// Any sizes and alignments, element by element: a thread takes a pair (d, d + R/2) of one row,
// or one dim past R, and finds its token's page and table row for itself. Bound by that: from some
// 256 tokens on 3 to 6 times the vector form's time (bf16 rows off 16 bytes, H32/KVH8/D128, 64 tokens
// 4.0 us and 4.0, 1024 24 and 7.9, 16384 386 and 85; 24 + 2 x 8 heads of 96 dims, 8192 tokens, 24
// rotated, off the chunks, 166 and, 32 rotated, 27). Copying 16-bit sources off 16 bytes first would
// pay from 5 M elements on (6 M 24.0 and 21.0 with the three copies, 24 M 88 and 43; 1.5 M 7.7 and
// 11.7), fp32 ones nowhere by much (24 M 84 and 101, 96 M 435 and 409).
template <typename ST, typename KT>
__global__ __launch_bounds__(kRwThreads) void rope_write_elt_kernel(const RopeWriteParams p) {
  const int half = p.R / 2;
  const int per_row = half + (p.D - p.R);
  const int rows = p.QH + 2 * p.KVH;
  const int64_t total = static_cast<int64_t>(p.batch) * p.tokens * rows * per_row;
  for (int64_t idx = static_cast<int64_t>(blockIdx.x) * kRwThreads + threadIdx.x; idx < total;
       idx += static_cast<int64_t>(gridDim.x) * kRwThreads) {
    const int i = static_cast<int>(idx % per_row);
    const int64_t rest = idx / per_row;
    const int r = static_cast<int>(rest % rows);
    const RwToken k = rw_token(p, rest / rows);
    const bool query = r < p.QH, value = r >= p.QH + p.KVH;
    if (!query && k.cache_off < 0) continue;
    const int h = query ? r : (value ? r - p.QH - p.KVH : r - p.QH);
    const int64_t* const ss = query ? p.q_src : (value ? p.v_src : p.k_src);
    const ST* const s = static_cast<const ST*>(query ? p.q : (value ? p.v : p.k)) + k.b * ss[0] +
                        k.t * ss[1] + h * ss[2];
    const bool pair = i < half;
    const int d0 = pair ? i : half + i, d1 = i + half;
    const float a = Elt<ST>::load(s + d0);
    const float b = pair ? Elt<ST>::load(s + d1) : 0.0f;
    float y0 = a, y1 = b;
    if (pair && !value) {
      const float* const ct = p.cos + k.table_off;
      const float* const st = p.sin + k.table_off;
      y0 = rope_mix(a, -b, ct[d0], st[d0]);
      y1 = rope_mix(b, a, ct[d1], st[d1]);
    }
    if (query) {
      ST* const d = static_cast<ST*>(p.q_out) + k.b * p.q_dst[0] + k.t * p.q_dst[1] + h * p.q_dst[2];
      Elt<ST>::store(d + d0, y0);
      if (pair) Elt<ST>::store(d + d1, y1);
    } else {
      KT* const d = static_cast<KT*>(value ? p.v_cache : p.k_cache) + k.cache_off + h * p.head_stride;
      Elt<KT>::store(d + d0, y0);
      if (pair) Elt<KT>::store(d + d1, y1);
    }
  }
}

// Elements of a vector: 16 bytes of the source.
template <typename ST>
constexpr int kRwVec = 16 / static_cast<int>(sizeof(ST));

template <typename ST, typename KT>
static bool rw_vec_ok(const RopeWriteParams& p) {
  constexpr int E = kRwVec<ST>;
  constexpr uintptr_t sa = E * sizeof(ST), da = E * sizeof(KT) >= 16 ? 16 : E * sizeof(KT);
  auto al = [](const void* q, uintptr_t a) { return reinterpret_cast<uintptr_t>(q) % a == 0; };
  for (int i = 0; i < 3; ++i)
    if (p.q_src[i] % E != 0 || p.k_src[i] % E != 0 || p.v_src[i] % E != 0 || p.q_dst[i] % E != 0)
      return false;
  return p.D % E == 0 && p.R % (2 * E) == 0 && p.D <= 2 * E * kWave && al(p.q, sa) && al(p.k, sa) &&
         al(p.v, sa) && al(p.q_out, sa) && al(p.cos, 16) && al(p.sin, 16) && al(p.k_cache, da) &&
         al(p.v_cache, da) && (p.blk_stride * sizeof(KT)) % da == 0 &&
         (p.slot_stride * sizeof(KT)) % da == 0 && (p.head_stride * sizeof(KT)) % da == 0;
}

template <typename ST, typename KT>
static hipError_t launch_rope_write_one(const RopeWriteParams& p_in, hipStream_t stream) {
  RopeWriteParams p = p_in;
  const int64_t tokens = static_cast<int64_t>(p.batch) * p.tokens;
  if (rw_vec_ok<ST, KT>(p)) {
    constexpr int E = kRwVec<ST>;
    p.items = ceil_div(p.D / E, 2);
    const int heads = kWave / p.items;
    const int most = ceil_div(p.QH + 2 * p.KVH, heads);
    // A token's rows are sliced over waves until the launch holds kRwWant of them.
    constexpr int64_t kRwWant = 4096;
    int64_t slices = (kRwWant + tokens - 1) / tokens;
    p.slices = static_cast<int>(slices < most ? slices : most);
    const int64_t blocks = (tokens * p.slices + kRwWaves - 1) / kRwWaves;
    if (blocks * kRwThreads < (int64_t(1) << 32)) {  // (a launch's threads are counted in 32 bits)
      hipLaunchKernelGGL((rope_write_vec_kernel<ST, KT, E>), dim3(static_cast<unsigned>(blocks)),
                         dim3(kRwThreads), 0, stream, p);
      return hipGetLastError();
    }
  }
  const int64_t total = tokens * (p.QH + 2 * p.KVH) * (p.D - p.R / 2);
  const int64_t blocks = (total + kRwThreads - 1) / kRwThreads;
  hipLaunchKernelGGL((rope_write_elt_kernel<ST, KT>),
                     dim3(static_cast<unsigned>(blocks < 65536 ? blocks : 65536)), dim3(kRwThreads),
                     0, stream, p);
  return hipGetLastError();
}

template <typename ST>
static hipError_t launch_rope_write_to(const RopeWriteParams& p, int kv_dtype, hipStream_t stream) {
  switch (kv_dtype) {
    case 0: return launch_rope_write_one<ST, float>(p, stream);
    case 1: return launch_rope_write_one<ST, _Float16>(p, stream);
    case 2: return launch_rope_write_one<ST, bf16_t>(p, stream);
    default: return launch_rope_write_one<ST, fp8_t>(p, stream);
  }
}

hipError_t launch_rope_write(const RopeWriteParams& p, int src_dtype, int kv_dtype,
                             hipStream_t stream) {
  switch (src_dtype) {
    case 0: return launch_rope_write_to<float>(p, kv_dtype, stream);
    case 1: return launch_rope_write_to<_Float16>(p, kv_dtype, stream);
    default: return launch_rope_write_to<bf16_t>(p, kv_dtype, stream);
  }
}

}  // namespace msattn
