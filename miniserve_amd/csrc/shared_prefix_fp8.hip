// Attention behind several shared prefixes over fp8 e4m3 caches.
#include "shared_prefix.h"

namespace msattn {

MSATTN_DEFINE_SHARED(bf16_t, fp8_t)
MSATTN_DEFINE_SHARED(_Float16, fp8_t)

}  // namespace msattn
