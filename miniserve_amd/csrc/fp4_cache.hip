// Keys and values into a 4-bit paged cache, and back (fp4_cache.h has the format).
//
//   write   cache[table[b, pos / bs], pos % bs] = quantise(src[b, t]),  pos = starts[b] + t
//   read    dst[b, t] = values of cache[table[b, pos / bs], pos % bs]
//
// One thread takes 8 elements of a row of K and of V: 16 bytes of a 16-bit row, 4 bytes of the
// cache. The four threads of a 32-element block are neighbours, so that the block's largest
// magnitude is two lane exchanges away.
#include "fp4_cache.h"

namespace msattn {

constexpr int kFp4Threads = 256;

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

// What a thread works on: 8 dims from 8 o of head h of token t of row b, and the tile and place
// of the token (tile < 0: a hole, or outside the table).
struct Fp4Item {
  int b, t, h, o;
  int64_t tile;  // byte offset of the tile in either cache
  int place;     // token within the tile
};

// Threads a token, a power of two up to the workgroup's; the grid's y covers what is left.
__host__ __device__ inline int fp4_lanes(int items) {
  int n = 4;
  while (n < items && n < kFp4Threads) n <<= 1;
  return n;
}

__device__ __forceinline__ bool fp4_item(const Fp4CacheParams& p, int lanes, int shift, Fp4Item* it) {
  const int tid = static_cast<int>(threadIdx.x);
  const int64_t row = (static_cast<int64_t>(blockIdx.x) << (8 - shift)) + (tid >> shift);
  const int item = static_cast<int>(blockIdx.y) * lanes + (tid & (lanes - 1));
  const int octets = p.D / 8;
  if (row >= static_cast<int64_t>(p.batch) * p.tokens || item >= p.KVH * octets) return false;
  it->b = fp4_quot(static_cast<int>(row), p.by_tokens);
  it->t = static_cast<int>(row) - it->b * p.tokens;
  it->h = fp4_quot(item, p.by_octets);
  it->o = item - it->h * octets;
  it->tile = -1;
  it->place = 0;
  const int64_t pos = static_cast<int64_t>(p.starts[it->b]) + it->t;
  if (pos < 0 || pos >= static_cast<int64_t>(p.W) * p.bs || pos >= (int64_t(1) << 31)) return true;
  const int pg = fp4_quot(static_cast<int>(pos), p.by_bs);
  const int phys = p.table[static_cast<int64_t>(it->b) * p.W + pg];
  if (phys < 0 || phys >= p.num_blocks) return true;
  const int in = static_cast<int>(pos) - pg * p.bs;
  it->tile = static_cast<int64_t>(phys) * p.blk_stride + static_cast<int64_t>(it->h) * p.head_stride +
             static_cast<int64_t>(in / kFp4Tile) * fp4_tile_bytes(p.D);
  it->place = in % kFp4Tile;
  return true;
}

__device__ __forceinline__ int64_t source_at(const int64_t (&st)[3], const Fp4Item& it) {
  return it.b * st[0] + it.t * st[1] + it.h * st[2] + 8 * it.o;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kFp4Threads) void write_fp4_kernel(const Fp4CacheParams p, int lanes,
                                                                int shift) {
  Fp4Item it;
  if (!fp4_item(p, lanes, shift, &it) || it.tile < 0) return;
  float k[8], v[8];
  load8<T, VEC>(static_cast<const T*>(p.k) + source_at(p.k_st, it), k);
  load8<T, VEC>(static_cast<const T*>(p.v) + source_at(p.v_st, it), v);
  uint32_t kb, vb;
  const uint32_t kw = quantise8(k, &kb), vw = quantise8(v, &vb);
  uint8_t* const kt = p.k_cache + it.tile;
  uint8_t* const vt = p.v_cache + it.tile;
  *reinterpret_cast<uint32_t*>(kt + it.place * (p.D / 2) + 4 * it.o) = kw;
  *reinterpret_cast<uint32_t*>(vt + 64 * it.o + 4 * it.place) = vw;
  if (it.o % 4 == 0) {
    const int at = 8 * p.D + 4 * it.o + it.place;
    kt[at] = static_cast<uint8_t>(kb);
    vt[at] = static_cast<uint8_t>(vb);
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kFp4Threads) void read_fp4_kernel(const Fp4CacheParams p, int lanes,
                                                               int shift) {
  Fp4Item it;
  if (!fp4_item(p, lanes, shift, &it)) return;
  float k[8], v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.0f;
  if (it.tile >= 0) {
    const uint8_t* const kt = p.k_cache + it.tile;
    const uint8_t* const vt = p.v_cache + it.tile;
    const int at = 8 * p.D + 16 * (it.o / 4) + it.place;
    widen8(*reinterpret_cast<const uint32_t*>(kt + it.place * (p.D / 2) + 4 * it.o), kt[at], k);
    widen8(*reinterpret_cast<const uint32_t*>(vt + 64 * it.o + 4 * it.place), vt[at], v);
  }
  store8<T, VEC>(static_cast<T*>(p.k) + source_at(p.k_st, it), k);
  store8<T, VEC>(static_cast<T*>(p.v) + source_at(p.v_st, it), v);
}

template <typename T, bool VEC>
static hipError_t launch_ops(const Fp4CacheParams& p, bool write, hipStream_t stream) {
  const int items = p.KVH * (p.D / 8);
  const int lanes = fp4_lanes(items);
  const int shift = __builtin_ctz(static_cast<unsigned>(lanes));
  const int64_t rows = static_cast<int64_t>(p.batch) * p.tokens, per = kFp4Threads / lanes;
  const dim3 grid(static_cast<unsigned>((rows + per - 1) / per),
                  static_cast<unsigned>((items + lanes - 1) / lanes));
  if (write)
    hipLaunchKernelGGL((write_fp4_kernel<T, VEC>), grid, dim3(kFp4Threads), 0, stream, p, lanes, shift);
  else
    hipLaunchKernelGGL((read_fp4_kernel<T, VEC>), grid, dim3(kFp4Threads), 0, stream, p, lanes, shift);
  return hipGetLastError();
}

template <bool VEC>
static hipError_t launch_types(const Fp4CacheParams& p, int dtype, bool write, hipStream_t stream) {
  switch (dtype) {
    case 0: return launch_ops<float, VEC>(p, write, stream);
    case 1: return launch_ops<_Float16, VEC>(p, write, stream);
    case 2: return launch_ops<bf16_t, VEC>(p, write, stream);
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
