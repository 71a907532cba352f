// Launches of the 4-bit cache's attention kernel for one query type (included by fp4_attn_*.hip).
#pragma once

#include "fp4_attn.h"

namespace msattn {

template <typename T, int DP, int CT>
static hipError_t fp4_launch(const Fp4Params& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(
      p.split ? p.shares : static_cast<int64_t>(p.batch) * p.rblocks * p.KVH));
  hipLaunchKernelGGL((fp4_attn_kernel<T, DP, CT>), grid, dim3(kFp4Threads), 0, stream, p);
  return hipGetLastError();
}

template <typename T, int DP>
static hipError_t fp4_launch_dim(const Fp4Params& p, int ct, hipStream_t stream) {
  if (ct == 1) return fp4_launch<T, DP, 1>(p, stream);
  if (ct == 2) return fp4_launch<T, DP, 2>(p, stream);
  return hipErrorNotSupported;
}

template <typename T>
hipError_t launch_fp4_attn(const Fp4Params& p, int ct, hipStream_t stream) {
  if (p.D <= 64) return fp4_launch_dim<T, 64>(p, ct, stream);
  if (p.D <= 128) return fp4_launch_dim<T, 128>(p, ct, stream);
  return fp4_launch_dim<T, 256>(p, ct, stream);
}

}  // namespace msattn
