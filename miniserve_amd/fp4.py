"""miniserve_amd.fp4 -- a paged K/V cache held in 4 bits.

17/32 of a byte an element (e2m1 elements, 32 of a row sharing a power of two: the MXFP4 format,
which gfx950 widens in one instruction), where a 16-bit cache (miniserve/attention.py:104-109) takes
2: a decode, which reads the whole cache once, has 3.76 times fewer bytes to read, and a card holds
3.76 times the contexts.

``allocate_fp4_cache`` makes the caches, ``write_kv_fp4`` quantises a step's keys and values into
them, ``paged_attention_fp4`` attends over them, and ``read_kv_fp4`` reads back the values that
positions stand for. ``PagedAttention(..., kv_dtype=torch.float4_e2m1fn_x2)`` does the same behind
its own methods. The layout is msattn.h's: uint8 [num_blocks, kv_heads, block_size / 16,
17 * head_dim / 2].
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _native as nat
from .attention import (_require_gpu, _workspace, block_table_i32, context_lens_i32, narrow_i32,
                        starts_i32)
from .rotary import _source, _spans, current, extent, on_16_bytes, on_device

TILE = 16     # tokens of a tile
BLOCK = 32    # elements that share a scale
_I64x3 = ctypes.c_int64 * 3
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


def _tile_bytes(head_dim: int) -> int:
    return 17 * head_dim // 2


def allocate_fp4_cache(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                       device: torch.device | str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """(k_cache, v_cache), each zeros [num_blocks, kv_heads, block_size / 16, 17 * head_dim / 2] of
    bytes, for pages of ``block_size`` tokens (a multiple of 16) and a ``head_dim`` that is a
    multiple of 32 up to 256."""
    if num_blocks <= 0 or num_kv_heads <= 0:
        raise ValueError("num_blocks and num_kv_heads must be positive")
    if block_size <= 0 or block_size % TILE:
        raise ValueError(f"block_size {block_size}: a 4-bit cache has pages of whole {TILE}-token "
                         "tiles")
    if head_dim <= 0 or head_dim % BLOCK or head_dim > nat.MAX_HEAD_DIM:
        raise ValueError(f"head_dim {head_dim}: a 4-bit cache takes multiples of {BLOCK} up to "
                         f"{nat.MAX_HEAD_DIM}")
    shape = (num_blocks, num_kv_heads, block_size // TILE, _tile_bytes(head_dim))
    return (torch.zeros(shape, dtype=torch.uint8, device=device),
            torch.zeros(shape, dtype=torch.uint8, device=device))


def is_fp4_cache(cache: torch.Tensor) -> bool:
    """Whether a cache tensor is one of ``allocate_fp4_cache``'s kind."""
    return cache.dtype == torch.uint8


def _cache_geometry(k_cache: torch.Tensor, v_cache: torch.Tensor) -> tuple[int, int, int, int]:
    """(num_blocks, kv_heads, block_size, head_dim) of a pair of 4-bit caches, which it checks."""
    if not (k_cache.is_cuda and v_cache.is_cuda):
        _require_gpu(k_cache, "k_cache")
        _require_gpu(v_cache, "v_cache")
    stride = k_cache.stride()
    if k_cache.ndim != 4 or k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8 or \
            k_cache.shape != v_cache.shape or stride != v_cache.stride():
        raise ValueError("k_cache and v_cache must share a uint8 [num_blocks, kv_heads, "
                         "block_size / 16, 17 * head_dim / 2] shape and strides")
    nb, KVH, tiles, nbytes = k_cache.shape
    D = nbytes * 2 // 17
    if nbytes != _tile_bytes(D) or D <= 0 or D % BLOCK or D > nat.MAX_HEAD_DIM:
        raise ValueError(f"a tile of {nbytes} bytes: a 4-bit cache has 17 * head_dim / 2, head_dim "
                         f"a multiple of {BLOCK} up to {nat.MAX_HEAD_DIM}")
    if nb == 0 or KVH == 0 or tiles == 0:
        raise ValueError("an empty cache")
    if stride[3] != 1 or tiles > 1 and stride[2] != nbytes or stride[0] % 16 or stride[1] % 16 or \
            k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16:
        raise ValueError("the tiles of a page and head must be contiguous, pages and heads on 16 "
                         "bytes")
    return nb, KVH, tiles * TILE, D


def write_kv_fp4(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_table, start=0) -> None:
    """Quantise ``k``/``v`` [batch, tokens, kv_heads, head_dim] (fp32, fp16 or bf16, any strides:
    the views of a fused projection are read where they lie) into the caches.

    Row b's token t goes to position start[b] + t (``start``: an int, one entry per row, or an int
    tensor); tokens on holes of the block table or outside it are not written. Each 32 elements of
    a row take the power of two 2^e for which the largest magnitude lies in (3.5, 7] 2^e, and go to
    the nearest of 0, 0.5, 1, 1.5, 2, 3, 4 and 6 times it (ties to the even code, at most 6), so
    that none is off by more than 2^e, a 3.5th of the largest; 32 elements with a NaN or an infinity
    among them read back as NaN. A row's bytes do not depend on what is written beside it. Two
    tokens of one call must not land in one slot: parts of either's rows may remain there.
    """
    nb, KVH, bs, D = _cache_geometry(k_cache, v_cache)
    dev, dtype = k_cache.device, k.dtype
    if not (k.is_cuda and v.is_cuda):
        _require_gpu(k, "k")
        _require_gpu(v, "v")
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError("k and v must both be [batch, tokens, kv_heads, head_dim]")
    B, T = k.shape[:2]
    if k.shape[2] != KVH or k.shape[3] != D:
        raise ValueError("k/v heads or head_dim do not match the cache")
    if v.dtype != dtype:
        raise ValueError("k and v must share a dtype")
    if dtype not in _TYPES:
        raise ValueError(f"unsupported dtype for a 4-bit cache: {dtype}")
    if v_cache.device != dev or k.device != dev or v.device != dev:
        raise ValueError("k, v and the caches must be on one device")
    if B == 0 or T == 0:
        return
    table = block_table_i32(block_table, dev)
    if table.shape[0] < B:
        raise ValueError("block_table has fewer rows than k")
    if table.shape[1] == 0:
        raise ValueError("block_table has no columns")
    if isinstance(start, torch.Tensor):
        start = narrow_i32(start)
    starts = starts_i32(start, B, dev)
    written = _spans((k_cache, v_cache))
    ks, vs = _source(k, written), _source(v, written)
    stride = k_cache.stride()
    status = on_device(
        dev, nat.lib().msattn_write_kv_fp4, ks.data_ptr(), _I64x3(*ks.stride()[:3]), vs.data_ptr(),
        _I64x3(*vs.stride()[:3]), k_cache.data_ptr(), v_cache.data_ptr(), stride[0], stride[1],
        table.data_ptr(), starts.data_ptr(), B, T, KVH, D, bs, nb, table.shape[1],
        nat.dtype_code(dtype))
    nat.check("msattn_write_kv_fp4", status)


def read_kv_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table, start, tokens: int, *,
                dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v), each [batch, tokens, kv_heads, head_dim] of ``dtype``: the values that positions
    start[b] .. start[b] + tokens - 1 of each block-table row stand for (``start``: an int, one
    entry per row, or an int tensor). fp32 and bf16 hold them exactly. Positions on holes, outside
    the table or below 0 give zeros; those past a row's context give whatever its pages hold.
    """
    nb, KVH, bs, D = _cache_geometry(k_cache, v_cache)
    dev = k_cache.device
    if v_cache.device != dev:
        raise ValueError("the caches must be on one device")
    if dtype not in _TYPES:
        raise ValueError(f"unsupported dtype for a 4-bit cache's values: {dtype}")
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    table = block_table_i32(block_table, dev)
    B, W = table.shape
    if W == 0:
        raise ValueError("block_table has no columns")
    k = torch.empty((B, tokens, KVH, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if k.numel() == 0:
        return k, v
    if isinstance(start, torch.Tensor):
        start = narrow_i32(start)
    starts = starts_i32(start, B, dev)
    stride = k_cache.stride()
    status = on_device(
        dev, nat.lib().msattn_read_kv_fp4, k_cache.data_ptr(), v_cache.data_ptr(), stride[0],
        stride[1], table.data_ptr(), starts.data_ptr(), k.data_ptr(), v.data_ptr(), B, tokens, KVH,
        D, bs, nb, W, nat.dtype_code(dtype))
    nat.check("msattn_read_kv_fp4", status)
    return k, v


def paged_attention_fp4(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        block_table, context_lens, *, causal: bool = True,
                        window: int | None = None, scale: float | None = None,
                        max_context: int | None = None, workspace: torch.Tensor | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention`` over a 4-bit cache: ``query`` [batch, q_len, heads, head_dim] (fp32, fp16
    or bf16), one query token a row, a few, or a chunk of a prompt, in one launch; the arguments as
    there. The cache's values enter exactly; an infinity or NaN reaches the queries that see its key
    alone. A view of the query in 16-byte rows is read where it lies. Nothing is read by the host
    where ``context_lens`` is a device tensor, so the call is safe to capture.
    """
    nb, KVH, bs, Dk = _cache_geometry(k_cache, v_cache)
    if not query.is_cuda:
        _require_gpu(query, "query")
    if query.ndim != 4:
        raise ValueError("query must be [batch, q_len, heads, head_dim]")
    B, q_len, H, D = query.shape
    if Dk != D:
        raise ValueError(f"head_dim mismatch: query {D}, cache {Dk}")
    if H == 0 or H % KVH:
        raise ValueError("num_heads must be a multiple of num_kv_heads")
    if query.dtype not in _TYPES:
        raise ValueError(f"unsupported dtype for a query over a 4-bit cache: {query.dtype}")
    if window is not None and window <= 0:
        raise ValueError("window must be positive")
    dev = query.device
    if k_cache.device != dev or v_cache.device != dev:
        raise ValueError("query and the caches must be on one device")
    table = block_table_i32(block_table, dev)
    if table.shape[0] != B:
        raise ValueError(f"block_table has {table.shape[0]} rows for a batch of {B}")
    W = table.shape[1]
    if W == 0:
        raise ValueError("block_table has no columns")
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or
                            out.device != dev or not out.is_contiguous()):
        raise ValueError("out must be contiguous, of the query's shape, dtype and device")
    if workspace is not None and (workspace.device != dev or not workspace.is_contiguous()):
        raise ValueError("workspace must be contiguous and on the query's device")
    with current(dev):
        lens, host_max = context_lens_i32(context_lens, dev, B)
    cap = W * bs
    if max_context is None:
        max_context = cap if host_max is None else host_max
    if host_max is not None and host_max > cap:
        raise ValueError(f"context length {host_max} exceeds the block table capacity {cap}")
    max_context = max(0, min(int(max_context), cap, 2 ** 31 - 1))
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    fresh = out is None
    if fresh:
        out = torch.empty((B, q_len, H, D), dtype=query.dtype, device=dev)
    if B == 0 or q_len == 0:
        return out
    given = None
    if out.data_ptr() % 16:  # (the kernel stores 16 bytes at once)
        given, out = out, torch.empty_like(out)
    q = query.resolve_neg() if query.is_neg() else query
    es = q.element_size()
    if q.stride(3) != 1 or any(s * es % 16 for s in q.stride()[:3]):
        q = q.contiguous()
    q = on_16_bytes(q)
    if q is query and not fresh:  # a wave reads its rows while another's are written
        (lo, hi), (olo, ohi) = extent(q), extent(out)
        if lo < ohi and olo < hi:
            q = q.clone(memory_format=torch.contiguous_format)
    lib = nat.lib()
    code = nat.dtype_code(q.dtype)
    ws_bytes = lib.msattn_fp4_workspace_bytes(B, q_len, H, KVH, D, max_context, code)
    if ws_bytes == 0:
        raise ValueError("unsupported attention geometry")
    if workspace is None or workspace.numel() * workspace.element_size() < ws_bytes:
        with current(dev):
            workspace = _workspace(dev, ws_bytes)
    stride = k_cache.stride()
    status = on_device(
        dev, lib.msattn_paged_attention_fp4, q.data_ptr(), _I64x3(*q.stride()[:3]),
        k_cache.data_ptr(), v_cache.data_ptr(), stride[0], stride[1], table.data_ptr(),
        lens.data_ptr(), out.data_ptr(), workspace.data_ptr(), ws_bytes, B, q_len, H, KVH, D, bs,
        nb, W, max_context, 1 if causal else 0, min(int(window or 0), 2 ** 31 - 1), float(scale),
        code)
    nat.check("msattn_paged_attention_fp4", status)
    return out if given is None else given.copy_(out)
