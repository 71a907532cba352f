// Attention behind several shared prefixes over bf16 and fp16 caches of the query's type.
#include "shared_prefix.h"

namespace msattn {

MSATTN_DEFINE_SHARED(bf16_t, bf16_t)
MSATTN_DEFINE_SHARED(_Float16, _Float16)

}  // namespace msattn
