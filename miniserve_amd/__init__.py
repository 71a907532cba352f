"""miniserve_amd -- MI355X-native paged attention for miniserve.

``PagedAttention`` keeps the interface of miniserve.attention.PagedAttention
and runs on hand-written gfx950 HIP kernels (libmsattn.so, C ABI in
include/msattn.h).
"""
from .attention import (PagedAttention, apply_rope, gather_kv, kernel_route, paged_attention,
                        paged_attention_append)
from .fp4 import allocate_fp4_cache, paged_attention_fp4, read_kv_fp4, write_kv_fp4
from .rotary import write_kv_rope
from .shared import paged_attention_shared

__all__ = ["PagedAttention", "allocate_fp4_cache", "apply_rope", "gather_kv", "kernel_route",
           "paged_attention", "paged_attention_append", "paged_attention_fp4",
           "paged_attention_shared", "read_kv_fp4", "write_kv_fp4", "write_kv_rope"]
