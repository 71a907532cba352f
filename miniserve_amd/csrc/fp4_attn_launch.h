// Launches of the 4-bit cache's attention kernel for one query type (included by fp4_attn_*.hip).
#pragma once

#include "fp4_attn.h"

namespace msattn {

template <typename T, int DP, int CT>
static hipError_t fp4_launch(const Fp4Params& p, hipStream_t stream) {
  const int64_t waves = p.split ? p.shares : static_cast<int64_t>(p.batch) * p.rblocks * p.KVH;
  const dim3 grid(static_cast<unsigned>((waves + kFp4Waves - 1) / kFp4Waves));
  hipLaunchKernelGGL((fp4_attn_kernel<T, DP, CT>), grid, dim3(64 * kFp4Waves), 0, stream, p);
  return hipGetLastError();
}

template <typename T, int DP>
static hipError_t fp4_launch_dim(const Fp4Params& p, int ct, hipStream_t stream) {
  if (ct == 1) return fp4_launch<T, DP, 1>(p, stream);
  if constexpr (DP < 256 && fp4_max_ct<T>() == 4)
    if (ct == 4) return fp4_launch<T, DP, 4>(p, stream);
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
