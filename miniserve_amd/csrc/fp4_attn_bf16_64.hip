// The 4-bit cache's attention kernel for bf16 queries and head sizes up to 64.
#include "fp4_attn_launch.h"

namespace msattn {
template hipError_t launch_fp4_attn<bf16_t, 64>(const Fp4Params&, int, int, int, hipStream_t);
}
