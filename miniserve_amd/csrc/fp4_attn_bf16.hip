// The 4-bit cache's attention kernel for bf16 queries.
#include "fp4_attn_launch.h"

namespace msattn {
template hipError_t launch_fp4_attn<bf16_t>(const Fp4Params&, int, hipStream_t);
}
