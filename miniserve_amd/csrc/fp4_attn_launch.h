// Launches of the 4-bit cache's attention kernel for one query type and head size (included by
// fp4_attn_*.hip).
#pragma once

#include "fp4_attn.h"

namespace msattn {

template <typename T, int DP, int CT, int WK, int WAY>
static hipError_t fp4_launch(const Fp4Params& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(WAY == kFp4List ? p.shares : 8 * p.xcd_units));
  hipLaunchKernelGGL((fp4_attn_kernel<T, DP, CT, WK, WAY>), grid, dim3(kFp4Threads), 0, stream, p);
  return hipGetLastError();
}

template <typename T, int DP, int CT>
static hipError_t fp4_launch_waves(const Fp4Params& p, int way, int wk, hipStream_t stream) {
  if constexpr (CT <= fp4_list_ct(fp4_parts<T>(), DP))
  {
    if (way == kFp4List) return fp4_launch<T, DP, CT, kFp4Waves, kFp4List>(p, stream);
    if (way == kFp4Parts) return fp4_launch<T, DP, CT, kFp4Waves, kFp4Parts>(p, stream);
  }
  if (way != kFp4Dealt) return hipErrorNotSupported;
  if constexpr (CT < 4)
    if (wk == 8) return fp4_launch<T, DP, CT, 8, kFp4Dealt>(p, stream);
  switch (wk) {
    case 1: return fp4_launch<T, DP, CT, 1, kFp4Dealt>(p, stream);
    case 2: return fp4_launch<T, DP, CT, 2, kFp4Dealt>(p, stream);
    case 4: return fp4_launch<T, DP, CT, 4, kFp4Dealt>(p, stream);
    default: return hipErrorNotSupported;
  }
}

template <typename T, int DP>
hipError_t launch_fp4_attn(const Fp4Params& p, int way, int ct, int wk, hipStream_t stream) {
  constexpr int most = fp4_max_ct(fp4_parts<T>(), DP);
  if (ct == 1) return fp4_launch_waves<T, DP, 1>(p, way, wk, stream);
  if constexpr (most >= 2)
    if (ct == 2) return fp4_launch_waves<T, DP, 2>(p, way, wk, stream);
  if constexpr (most >= 4)
    if (ct == 4) return fp4_launch_waves<T, DP, 4>(p, way, wk, stream);
  return hipErrorNotSupported;
}

}  // namespace msattn
