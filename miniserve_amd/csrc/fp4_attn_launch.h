// Launches of the 4-bit cache's attention kernel for one query type and head size (included by
// fp4_attn_*.hip).
#pragma once

#include "fp4_attn.h"

namespace msattn {

template <typename T, int DP, int CT, int WK>
static hipError_t fp4_launch(const Fp4Params& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.split ? p.shares : 8 * p.xcd_units));
  hipLaunchKernelGGL((fp4_attn_kernel<T, DP, CT, WK>), grid, dim3(kFp4Threads), 0, stream, p);
  return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch_fp4_attn(const Fp4Params& p, int ct, int wk, hipStream_t stream) {
  if (ct == 1) return fp4_launch<T, DP, 1, 8>(p, stream);
  if constexpr (fp4_max_ct<T, DP>() == 4) {
    if (ct == 4 && wk == 1) return fp4_launch<T, DP, 4, 1>(p, stream);
    if (ct == 4 && wk == 2) return fp4_launch<T, DP, 4, 2>(p, stream);
    if (ct == 4) return fp4_launch<T, DP, 4, 4>(p, stream);
  }
  switch (wk) {
    case 1: return fp4_launch<T, DP, 2, 1>(p, stream);
    case 2: return fp4_launch<T, DP, 2, 2>(p, stream);
    case 4: return fp4_launch<T, DP, 2, 4>(p, stream);
    default: return fp4_launch<T, DP, 2, 8>(p, stream);
  }
}

}  // namespace msattn
