// The 4-bit cache's attention kernel for f16 queries.
#include "fp4_attn_launch.h"

namespace msattn {
template hipError_t launch_fp4_attn<_Float16>(const Fp4Params&, int, hipStream_t);
}
