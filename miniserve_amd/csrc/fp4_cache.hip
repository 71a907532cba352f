// Keys and values into a 4-bit paged cache, and back (fp4_cache.h has the format).
//
//   write   cache[table[b, pos / bs], pos % bs] = quantise(src[b, t]),  pos = starts[b] + t
//   read    dst[b, t] = values of cache[table[b, pos / bs], pos % bs]
//
// A wave takes one tile (16 tokens of one head) of K and of V, four lanes a token: in step j lane
// (t, q) = (l / 4, l % 4) has dims 32 j + 8 q .. + 7 of token t, 16 bytes of a 16-bit row and 4 of the
// cache, so that a block's largest magnitude is two lane exchanges away. Rows move in pieces of 64
// bytes; values' tiles in whole lines, since octet 4 j + q lies at 64 (4 j + q) + 4 t; keys' too, once
// the four lanes of a token have exchanged their words of four steps. (A thread for each 8 elements,
// row by row, wrote the values' words 64 bytes apart: 4 x 8191 tokens of 8 x 128 bf16 in 51 us.)
#include "fp4_cache.h"

namespace msattn {

// Eight elements of a row in fp32. VEC: 16-byte accesses.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (VEC) {
    constexpr int N = Chunk<T>::kElems;
#pragma unroll
    for (int i = 0; i < 8 / N; ++i)
      Chunk<T>::unpack(*reinterpret_cast<const uint4*>(p + i * N), x + i * N);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elt<T>::load(p + i);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) Elt<T>::store(p + i, x[i]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = Chunk<T>::pack(x);
  }
}

// Largest of the values of the lane's aligned group of four lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  const uint32_t a = static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0xB1, 0xF, 0xF, true));
  x = x > a ? x : a;
  const uint32_t b = static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), 0x4E, 0xF, 0xF, true));
  return x > b ? x : b;
}

// The scale byte of a block from the bits of its largest magnitude: adding 0x1fffff carries into
// the exponent where the significand is above 1.75.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return kFp4NaN;
  const int e = static_cast<int>((top + 0x1fffffu) >> 23) - 2;
  return static_cast<uint32_t>(e < 1 ? 1 : (e > 252 ? 252 : e));
}

// This thread's 8 elements as 4 bytes, and the block's scale byte. v_cvt_scalef32_pk_fp4_f32
// divides by the scale, rounds to the nearest even code and saturates at 6.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t* byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __float_as_uint(x[i]) & 0x7fffffffu;
    top = a > top ? a : top;
  }
  *byte = scale_byte(quad_max(top));
  const float s = fp4_scale(*byte);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return *byte == kFp4NaN ? 0u : w;
}

__device__ __forceinline__ void widen8(uint32_t w, uint32_t byte, float (&x)[8]) {
  const float s = fp4_scale(byte);
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0);
  const f2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1);
  const f2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2);
  const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
  const float y[8] = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = byte == kFp4NaN ? __uint_as_float(0x7fc00000u) : y[i];
}

// What a wave works on: head h and the tokens of one tile of row b, and where the tile lies (at < 0:
// a hole, or outside the table).
struct Fp4Item {
  int b, h;
  int t;       // the lane's token (in the call's rows)
  bool live;   // which is one of the call's
  int64_t at;  // byte offset of the tile in either cache
};

__device__ __forceinline__ bool fp4_item(const Fp4CacheParams& p, Fp4Item* it) {
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int64_t i64 = static_cast<int64_t>(blockIdx.x) * (kFp4CacheThreads / 64) + wave;
  if (i64 >= p.items) return false;
  const int i = static_cast<int>(i64);
  const int bk = fp4_quot(i, p.by_heads);  // (head fastest: its neighbours' rows are the memory's)
  it->h = i - bk * p.KVH;
  it->b = fp4_quot(bk, p.by_tiles);
  const int k = bk - it->b * p.tiles;      // the row's tile, from the one its first token lies in
  const int64_t start = p.starts[it->b];
  const int64_t first = ((start >> 4) + k) << 4;  // the tile's first position
  it->t = static_cast<int>(first - start) + (static_cast<int>(threadIdx.x) & 63) / 4;
  it->live = it->t >= 0 && it->t < p.tokens;
  it->at = -1;
  if (first < 0 || first >= static_cast<int64_t>(p.W) * p.bs || first >= (int64_t(1) << 31)) return true;
  const int pg = fp4_quot(static_cast<int>(first), p.by_bs);
  const int phys = __builtin_amdgcn_readfirstlane(p.table[static_cast<int64_t>(it->b) * p.W + pg]);
  if (phys < 0 || phys >= p.num_blocks) return true;
  it->at = static_cast<int64_t>(phys) * p.blk_stride + static_cast<int64_t>(it->h) * p.head_stride +
           static_cast<int64_t>((static_cast<int>(first) - pg * p.bs) / kFp4Tile) * fp4_tile_bytes(p.D);
  return true;
}

// Words x[j] of lanes q = 0 .. 3 of a quad, transposed: x[j] of lane q becomes x[q] of lane j.
__device__ __forceinline__ void quad_transpose(uint32_t (&x)[4], int q) {
  auto swapped = [](uint32_t v, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v),
                                                             decltype(ctrl)::value, 0xF, 0xF, true));
  };
  using X1 = std::integral_constant<int, 0xB1>;  // lane q ^ 1
  using X2 = std::integral_constant<int, 0x4E>;  // lane q ^ 2
#pragma unroll
  for (int j = 0; j < 4; j += 2) {  // the off-diagonal words of each 2 x 2, then the 2 x 2s
    const uint32_t send = q & 1 ? x[j] : x[j + 1];
    const uint32_t got = swapped(send, X1{});
    if (q & 1) x[j] = got;
    else x[j + 1] = got;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t send = q & 2 ? x[j] : x[j + 2];
    const uint32_t got = swapped(send, X2{});
    if (q & 2) x[j] = got;
    else x[j + 2] = got;
  }
}

template <typename T, bool VEC, int NB>
__global__ __launch_bounds__(kFp4CacheThreads) void write_fp4_kernel(const Fp4CacheParams p) {
  Fp4Item it;
  if (!fp4_item(p, &it) || it.at < 0 || !it.live) return;  // (a token's four lanes as one)
  const int lane = static_cast<int>(threadIdx.x) & 63, t = lane >> 2, q = lane & 3;
  const T* const kp = static_cast<const T*>(p.k) + it.b * p.k_st[0] + it.t * p.k_st[1] + it.h * p.k_st[2] + 8 * q;
  const T* const vp = static_cast<const T*>(p.v) + it.b * p.v_st[0] + it.t * p.v_st[1] + it.h * p.v_st[2] + 8 * q;
  uint8_t* const kt = p.k_cache + it.at;
  uint8_t* const vt = p.v_cache + it.at;
  uint32_t kw[NB], kb[NB], vw[NB], vb[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    float x[8];
    load8<T, VEC>(kp + 32 * j, x);
    kw[j] = quantise8(x, &kb[j]);
    load8<T, VEC>(vp + 32 * j, x);
    vw[j] = quantise8(x, &vb[j]);
  }
#pragma unroll
  for (int j = 0; j + 4 <= NB; j += 4) {
    uint32_t x[4] = {kw[j], kw[j + 1], kw[j + 2], kw[j + 3]};
    quad_transpose(x, q);  // lane q: all of block j + q
    *reinterpret_cast<uint4*>(kt + t * (16 * NB) + 16 * (j + q)) = make_uint4(x[0], x[1], x[2], x[3]);
  }
#pragma unroll
  for (int j = NB / 4 * 4; j < NB; ++j)
    *reinterpret_cast<uint32_t*>(kt + t * (16 * NB) + 16 * j + 4 * q) = kw[j];
#pragma unroll
  for (int j = 0; j < NB; ++j)
    *reinterpret_cast<uint32_t*>(vt + 64 * (4 * j + q) + 4 * t) = vw[j];
#pragma unroll
  for (int j = 0; j < NB; ++j) {  // (lane j % 4 stores block j's bytes)
    if (q != j % 4) continue;
    kt[256 * NB + 16 * j + t] = static_cast<uint8_t>(kb[j]);
    vt[256 * NB + 16 * j + t] = static_cast<uint8_t>(vb[j]);
  }
}

// Lanes l and l + 4 (bit 2 of l clear) hold dims 32 j .. (a) and 32 (j + 1) .. (b) of two tokens in
// turn; afterwards l's a and l + 4's a are the first token's 64 dims, and their b the second's.
__device__ __forceinline__ void swap_halves(uint4& a, uint4& b) {
  const bool second = (static_cast<int>(threadIdx.x) & 4) != 0;
  const auto one = [second](uint32_t& x, uint32_t& y) {
    const int send = static_cast<int>(second ? x : y);
    const uint32_t from_next =
        static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, send, 0x104, 0xF, 0xF, true));
    const uint32_t from_last =
        static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, send, 0x114, 0xF, 0xF, true));
    const uint32_t kept = second ? y : x;
    x = second ? from_last : kept;
    y = second ? kept : from_next;
  };
  one(a.x, b.x);
  one(a.y, b.y);
  one(a.z, b.z);
  one(a.w, b.w);
}

template <typename T, bool VEC, int NB>
__global__ __launch_bounds__(kFp4CacheThreads) void read_fp4_kernel(const Fp4CacheParams p) {
  Fp4Item it;
  if (!fp4_item(p, &it)) return;  // (a wave at a time; lanes without a token only pass words on)
  const int lane = static_cast<int>(threadIdx.x) & 63, t = lane >> 2, q = lane & 3;
  const int64_t at = it.b * p.k_st[0] + it.t * p.k_st[1] + it.h * p.k_st[2] + 8 * q;
  uint32_t kw[NB], kb[NB], vw[NB], vb[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) kw[j] = vw[j] = kb[j] = vb[j] = 0;
  if (it.at >= 0) {
    const uint8_t* const kt = p.k_cache + it.at;
    const uint8_t* const vt = p.v_cache + it.at;
#pragma unroll
    for (int j = 0; j + 4 <= NB; j += 4) {
      const uint4 w = *reinterpret_cast<const uint4*>(kt + t * (16 * NB) + 16 * (j + q));
      uint32_t x[4] = {w.x, w.y, w.z, w.w};
      quad_transpose(x, q);  // lane q: octet q of blocks j .. j + 3
#pragma unroll
      for (int i = 0; i < 4; ++i) kw[j + i] = x[i];
    }
#pragma unroll
    for (int j = NB / 4 * 4; j < NB; ++j)
      kw[j] = *reinterpret_cast<const uint32_t*>(kt + t * (16 * NB) + 16 * j + 4 * q);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      vw[j] = *reinterpret_cast<const uint32_t*>(vt + 64 * (4 * j + q) + 4 * t);
      kb[j] = kt[256 * NB + 16 * j + t];
      vb[j] = vt[256 * NB + 16 * j + t];
    }
  }
  // Rows of 16-bit elements leave two blocks a step, so that eight lanes write a line of 128 bytes at
  // once: with four lanes' 64 bytes a store (what other types and a last odd block do), answers
  // larger than a cache were read and written back a half line at a time (134 MB in 52.5 us, now
  // 37.2; 67 MB in 29.5, now 20.3; the same below 34 MB). Stores past the caches were as fast here, and
  // cost the answer's reader more than that (134 MB read and reduced in 136 us, against 109).
  constexpr bool kPairs = VEC && sizeof(T) == 2;
  constexpr int kPaired = kPairs ? NB / 2 * 2 : 0;
  T* const out[2] = {static_cast<T*>(p.k) + at, static_cast<T*>(p.v) + at};
  if constexpr (kPairs) {
    const int second = t & 1;
    const int64_t from = 32 * second - (second ? p.k_st[1] : 0);
    const int t0 = it.t - second;
    const bool live0 = t0 >= 0 && t0 < p.tokens, live1 = t0 + 1 >= 0 && t0 + 1 < p.tokens;
#pragma unroll
    for (int of = 0; of < 2; ++of)
#pragma unroll
      for (int j = 0; j < kPaired; j += 2) {
        float x[8], y[8];
        widen8(of ? vw[j] : kw[j], of ? vb[j] : kb[j], x);
        widen8(of ? vw[j + 1] : kw[j + 1], of ? vb[j + 1] : kb[j + 1], y);
        uint4 a = Chunk<T>::pack(x), b = Chunk<T>::pack(y);
        swap_halves(a, b);
        T* const o = out[of] + from + 32 * j;
        if (live0) *reinterpret_cast<uint4*>(o) = a;
        if (live1) *reinterpret_cast<uint4*>(o + p.k_st[1]) = b;
      }
  }
  if (!it.live) return;
#pragma unroll
  for (int j = kPaired; j < NB; ++j) {
    float x[8];
    widen8(kw[j], kb[j], x);
    store8<T, VEC>(out[0] + 32 * j, x);
    widen8(vw[j], vb[j], x);
    store8<T, VEC>(out[1] + 32 * j, x);
  }
}

template <typename T, bool VEC, int NB>
static hipError_t launch_ops(const Fp4CacheParams& p, bool write, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(fp4_cache_workgroups(p.items)));
  if (write)
    hipLaunchKernelGGL((write_fp4_kernel<T, VEC, NB>), grid, dim3(kFp4CacheThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((read_fp4_kernel<T, VEC, NB>), grid, dim3(kFp4CacheThreads), 0, stream, p);
  return hipGetLastError();
}

template <typename T, bool VEC>
static hipError_t launch_blocks(const Fp4CacheParams& p, bool write, hipStream_t stream) {
  switch (p.D / kFp4Block) {
    case 1: return launch_ops<T, VEC, 1>(p, write, stream);
    case 2: return launch_ops<T, VEC, 2>(p, write, stream);
    case 3: return launch_ops<T, VEC, 3>(p, write, stream);
    case 4: return launch_ops<T, VEC, 4>(p, write, stream);
    case 5: return launch_ops<T, VEC, 5>(p, write, stream);
    case 6: return launch_ops<T, VEC, 6>(p, write, stream);
    case 7: return launch_ops<T, VEC, 7>(p, write, stream);
    case 8: return launch_ops<T, VEC, 8>(p, write, stream);
    default: return hipErrorNotSupported;
  }
}

template <bool VEC>
static hipError_t launch_types(const Fp4CacheParams& p, int dtype, bool write, hipStream_t stream) {
  switch (dtype) {
    case 0: return launch_blocks<float, VEC>(p, write, stream);
    case 1: return launch_blocks<_Float16, VEC>(p, write, stream);
    case 2: return launch_blocks<bf16_t, VEC>(p, write, stream);
    default: return hipErrorNotSupported;
  }
}

hipError_t launch_write_fp4(const Fp4CacheParams& p, int src_dtype, hipStream_t stream) {
  return p.vec ? launch_types<true>(p, src_dtype, true, stream)
               : launch_types<false>(p, src_dtype, true, stream);
}

hipError_t launch_read_fp4(const Fp4CacheParams& p, int dst_dtype, hipStream_t stream) {
  return p.vec ? launch_types<true>(p, dst_dtype, false, stream)
               : launch_types<false>(p, dst_dtype, false, stream);
}

}  // namespace msattn
