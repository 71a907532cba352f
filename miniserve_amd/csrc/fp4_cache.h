// A paged K/V cache held in 4 bits (gfx950): its layout, and the kernels' parameters.
//
// Elements are e2m1 (a sign and 0, 0.5, 1, 1.5, 2, 3, 4, 6); each 32 of a row share a power of
// two, held as its exponent + 127 in a byte (the OCP microscaling format MXFP4, which gfx950
// widens and rounds in one instruction each). For a block whose largest magnitude is a the
// power is the one that puts a / 2^e in (3.5, 7]: a rounds to 4 or 6, off by at most a fifth of it
// (5 to 4), and no element by more than 2^e.
// (The rms error of normal values is 0.1119 of theirs, against 0.1149 for the exponent of a alone
// and 0.1155 for the smallest power that saturates nothing.) Elements round to the nearest, ties to
// the even code. The bytes 1 .. 252 are used, so that both the power and 6 times it are normal in
// fp32 and bf16; past 7 2^125 a saturates at 6 2^125, below 3.5 2^-126 it takes 2^-126. A block with a NaN or an infinity has the byte 255: all of it reads as NaN.
//
// A cache is uint8 [num_blocks, kv_heads, block_size / 16, 17 D / 2]: one tile, contiguous, for 16
// tokens of one head, its 8 D bytes of elements and then its scales as [D / 32][16 tokens]. Two
// elements share a byte, the earlier dim low. The elements lie as the attention kernel's lanes take
// them, 16 bytes a lane, 1 KiB a wave at D = 128:
//   keys    [16 tokens][D / 2]             a lane takes 32 dims of a token
//   values  [D / 8][16 tokens][4]          a lane takes 8 dims of 4 tokens
// (in the 16-bit caches' order a head's rows of 4-bit elements would be 64 bytes each, a page's
// stride apart, half a cache line).
#pragma once

#include "common.h"

namespace msattn {

constexpr int kFp4Tile = 16;    // tokens of a tile
constexpr int kFp4Block = 32;   // elements that share a scale
constexpr int kFp4MaxDim = 256;
constexpr int kFp4NaN = 255;    // the scale byte of a block that reads as NaN

__host__ __device__ constexpr int fp4_tile_bytes(int D) { return 17 * D / 2; }

// The power of two of a scale byte (NaN for 255 is left to the caller; 2^127 + 1 is no byte of
// this library's).
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Division of x < 2^31 by a constant of the call: with s = ceil(log2 d) and m = ceil(2^(31+s) / d),
// x m 2^-(31+s) exceeds x / d by less than 1 / d, so its integer part is the quotient.
struct Fp4Div {
  uint32_t m;
  int s;
};
inline Fp4Div fp4_div(uint32_t d) {
  Fp4Div f;
  f.s = 0;
  while ((uint64_t(1) << f.s) < d) ++f.s;
  f.m = static_cast<uint32_t>(((uint64_t(1) << (31 + f.s)) + d - 1) / d);
  return f;
}
__device__ __forceinline__ int fp4_quot(int x, Fp4Div f) {
  return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(x), f.m) >> f.s);
}

// msattn_write_kv_fp4 and msattn_read_kv_fp4.
struct Fp4CacheParams {
  uint8_t* k_cache;
  uint8_t* v_cache;
  void* k;  // written from, or read into
  void* v;
  const int32_t* table;
  const int32_t* starts;
  int64_t blk_stride, head_stride;  // bytes
  int64_t k_st[3], v_st[3];         // batch, token and head strides of k and v (elements)
  int batch, tokens, KVH, D, bs, num_blocks, W;
  int vec;                          // rows of k and v on 16 bytes
  int tiles;                        // that a row's tokens may touch
  int64_t items;                    // rows x tiles x heads: a wave each
  Fp4Div by_tiles, by_heads, by_bs;
};

constexpr int kFp4CacheThreads = 256;  // of a workgroup of theirs
constexpr int64_t fp4_cache_workgroups(int64_t items) {
  return (items + kFp4CacheThreads / 64 - 1) / (kFp4CacheThreads / 64);
}

hipError_t launch_write_fp4(const Fp4CacheParams& p, int src_dtype, hipStream_t stream);
hipError_t launch_read_fp4(const Fp4CacheParams& p, int dst_dtype, hipStream_t stream);

}  // namespace msattn
