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

import math

import torch

from . import _native as nat
from .attention import (_require_gpu, _workspace, _workspaces, block_table_i32,
                        context_lens_i32, narrow_i32, starts_i32)
from .rotary import current, extent, on_device

TILE = 16     # tokens of a tile
BLOCK = 32    # elements that share a scale
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


def cache_geometry(k_cache: torch.Tensor, v_cache: torch.Tensor
                    ) -> tuple[int, int, int, int, int, tuple]:
    """(device index, num_blocks, kv_heads, block_size, head_dim, strides) of a pair of 4-bit
    caches, which it checks (all but what the library's entry points check)."""
    at, shape, stride = k_cache.get_device(), k_cache.shape, k_cache.stride()
    if at < 0 or v_cache.get_device() != at:
        _require_gpu(k_cache, "k_cache")
        _require_gpu(v_cache, "v_cache")
        raise ValueError("the caches must be on one device")
    if len(shape) != 4 or shape != v_cache.shape or stride != v_cache.stride() or \
            k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8:
        raise ValueError("k_cache and v_cache must share a uint8 [num_blocks, kv_heads, "
                         "block_size / 16, 17 * head_dim / 2] shape and strides")
    nb, KVH, tiles, nbytes = shape
    D = nbytes * 2 // 17
    if nbytes != _tile_bytes(D) or D <= 0 or D % BLOCK or D > nat.MAX_HEAD_DIM:
        raise ValueError(f"a tile of {nbytes} bytes: a 4-bit cache has 17 * head_dim / 2, head_dim "
                         f"a multiple of {BLOCK} up to {nat.MAX_HEAD_DIM}")
    if not (nb and KVH and tiles):
        raise ValueError("an empty cache")
    if stride[3] != 1 or stride[2] != nbytes and tiles > 1:
        raise ValueError("the tiles of a page and head must be contiguous")
    return at, nb, KVH, tiles * TILE, D, stride


def _check(fn: str, status: int, k_cache: torch.Tensor, v_cache: torch.Tensor) -> None:
    """nat.check, naming what a refusal of the caches is about."""
    if status == nat.ERR_INVALID_ARG and (
            any(x % 16 for x in k_cache.stride()[:2]) or k_cache.data_ptr() % 16 or
            v_cache.data_ptr() % 16):
        raise ValueError(f"{fn}: a 4-bit cache's pages and heads lie on 16 bytes")
    nat.check(fn, status)


def write_kv_fp4(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_table, start=0) -> None:
    """Quantise ``k``/``v`` [batch, tokens, kv_heads, head_dim] (fp32, fp16 or bf16, any strides:
    the views of a fused projection are read where they lie) into the caches.

    Row b's token t goes to position start[b] + t (``start``: an int, one entry per row, or an int
    tensor); tokens on holes of the block table or outside it are not written. Each 32 elements of
    a row take the power of two 2^e for which the largest magnitude lies in (3.5, 7] 2^e (-126 <= e
    <= 125), and go to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4 and 6 times it (ties to the even code,
    at most 6), so that none is off by more than 2^e, a 3.5th of the largest, where that is from
    4.1e-38 to 2.9e38 (larger ones saturate at 6 2^125); 32 elements with a NaN or an infinity
    among them read back as NaN. A row's bytes do not depend on what is written beside it. Two
    tokens of one call must not land in one slot: parts of either's rows may remain there.
    """
    at, nb, KVH, bs, D, stride = cache_geometry(k_cache, v_cache)
    if k.get_device() != at or v.get_device() != at:
        _require_gpu(k, "k")
        _require_gpu(v, "v")
        raise ValueError("k, v and the caches must be on one device")
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or shape != v.shape:
        raise ValueError("k and v must both be [batch, tokens, kv_heads, head_dim]")
    B, T = shape[:2]
    if shape[2] != KVH or shape[3] != D:
        raise ValueError("k/v heads or head_dim do not match the cache")
    if v.dtype != dtype:
        raise ValueError("k and v must share a dtype")
    if dtype not in _TYPES:
        raise ValueError(f"unsupported dtype for a 4-bit cache: {dtype}")
    if B == 0 or T == 0:
        return
    dev = k_cache.device
    table = block_table_i32(block_table, dev)
    rows, W = table.shape
    if rows < B:
        raise ValueError("block_table has fewer rows than k")
    if W == 0:
        raise ValueError("block_table has no columns")
    if isinstance(start, torch.Tensor):
        start = narrow_i32(start)
    starts = starts_i32(start, B, dev)
    ks, vs = k.stride(), v.stride()
    fn, code = nat.lib().msattn_write_kv_fp4, nat.DTYPE_CODES[dtype]
    if ks[3] != 1 or vs[3] != 1 or k.is_neg() or v.is_neg():
        status = nat.ERR_OVERLAP
    else:
        status = on_device(
            dev, fn, k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2],
            k_cache.data_ptr(), v_cache.data_ptr(), stride[0], stride[1], table.data_ptr(),
            starts.data_ptr(), B, T, KVH, D, bs, nb, W, code)
    if status == nat.ERR_OVERLAP:  # rows that cannot be read where they lie: a copy
        with current(dev):
            k, v = (x.resolve_neg().clone(memory_format=torch.contiguous_format) for x in (k, v))
        ks = k.stride()
        status = on_device(
            dev, fn, k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), ks[0], ks[1], ks[2],
            k_cache.data_ptr(), v_cache.data_ptr(), stride[0], stride[1], table.data_ptr(),
            starts.data_ptr(), B, T, KVH, D, bs, nb, W, code)
    if status:
        _check("msattn_write_kv_fp4", status, k_cache, v_cache)


def read_kv_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table, start, tokens: int, *,
                dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v), each [batch, tokens, kv_heads, head_dim] of ``dtype``: the values that positions
    start[b] .. start[b] + tokens - 1 of each block-table row stand for (``start``: an int, one
    entry per row, or an int tensor). fp32 and bf16 hold them exactly. Positions on holes, outside
    the table or below 0 give zeros; those past a row's context give whatever its pages hold.
    """
    _, nb, KVH, bs, D, stride = cache_geometry(k_cache, v_cache)
    if dtype not in _TYPES:
        raise ValueError(f"unsupported dtype for a 4-bit cache's values: {dtype}")
    tokens = int(tokens)
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    dev = k_cache.device
    table = block_table_i32(block_table, dev)
    B, W = table.shape
    if W == 0:
        raise ValueError("block_table has no columns")
    k, v = torch.empty((2, B, tokens, KVH, D), dtype=dtype, device=dev).unbind(0)
    if B == 0 or tokens == 0:
        return k, v
    if isinstance(start, torch.Tensor):
        start = narrow_i32(start)
    starts = starts_i32(start, B, dev)
    status = on_device(
        dev, nat.lib().msattn_read_kv_fp4, k_cache.data_ptr(), v_cache.data_ptr(), stride[0],
        stride[1], table.data_ptr(), starts.data_ptr(), k.data_ptr(), v.data_ptr(), B, tokens, KVH,
        D, bs, nb, W, nat.DTYPE_CODES[dtype])
    if status:
        _check("msattn_read_kv_fp4", status, k_cache, v_cache)
    return k, v


def _kept_workspace(dev: torch.device, index: int) -> torch.Tensor | None:
    """The workspace that calls on `dev`'s current stream share (None where there is none yet, and
    under capture, where a graph gets one of its own)."""
    if torch._C._cuda_getDevice() != index or torch.cuda.is_current_stream_capturing():
        return None
    return _workspaces.get((index, nat.stream_handle(dev)))


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
    at, nb, KVH, bs, Dk, stride = cache_geometry(k_cache, v_cache)
    if query.get_device() != at:
        _require_gpu(query, "query")
        raise ValueError("query and the caches must be on one device")
    shape, dtype = query.shape, query.dtype
    if len(shape) != 4:
        raise ValueError("query must be [batch, q_len, heads, head_dim]")
    B, q_len, H, D = shape
    if Dk != D:
        raise ValueError(f"head_dim mismatch: query {D}, cache {Dk}")
    if H == 0 or H % KVH:
        raise ValueError("num_heads must be a multiple of num_kv_heads")
    if dtype not in _TYPES:
        raise ValueError(f"unsupported dtype for a query over a 4-bit cache: {dtype}")
    if window is not None and window <= 0:
        raise ValueError("window must be positive")
    dev = query.device
    table = block_table_i32(block_table, dev)
    rows, W = table.shape
    if rows != B:
        raise ValueError(f"block_table has {rows} rows for a batch of {B}")
    if W == 0:
        raise ValueError("block_table has no columns")
    if workspace is not None and (workspace.device != dev or not workspace.is_contiguous()):
        raise ValueError("workspace must be contiguous and on the query's device")
    if isinstance(context_lens, torch.Tensor):
        context_lens = narrow_i32(context_lens)
    lens, host_max = context_lens_i32(context_lens, dev, B)
    cap = W * bs
    if max_context is None:
        max_context = cap if host_max is None else host_max
    if host_max is not None and host_max > cap:
        raise ValueError(f"context length {host_max} exceeds the block table capacity {cap}")
    max_context = max(0, min(int(max_context), cap, 2 ** 31 - 1))
    given = None  # an output that the kernel, which stores 16 bytes at once, does not write itself
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != shape or out.dtype != dtype or out.device != dev or not out.is_contiguous():
        raise ValueError("out must be contiguous, of the query's shape, dtype and device")
    else:
        (lo, hi), (olo, ohi) = extent(query), extent(out)
        if lo < ohi and olo < hi:  # a wave reads its rows while another's are written
            query = query.clone()
        if olo % 16:
            given, out = out, torch.empty_like(out)
    if B == 0 or q_len == 0:
        return out if given is None else given
    qs = query.stride()
    es = 16 // query.element_size()
    if qs[3] != 1 or qs[0] % es or qs[1] % es or qs[2] % es or query.data_ptr() % 16 or \
            query.is_neg():
        query = query.resolve_neg().clone(memory_format=torch.contiguous_format)
        qs = query.stride()
    lib, code = nat.lib(), nat.DTYPE_CODES[dtype]
    args = (query.data_ptr(), qs[0], qs[1], qs[2], k_cache.data_ptr(), v_cache.data_ptr(),
            stride[0], stride[1], table.data_ptr(), lens.data_ptr(), out.data_ptr())
    sizes = (B, q_len, H, KVH, D, bs, nb, W, max_context, 1 if causal else 0,
             min(window or 0, 2 ** 31 - 1), 1.0 / math.sqrt(D) if scale is None else float(scale),
             code)
    status, call = nat.ERR_WORKSPACE, lib.msattn_paged_attention_fp4
    if workspace is None:  # the stream's, as large as earlier calls needed it
        workspace = _kept_workspace(dev, at)
    if workspace is not None:
        status = on_device(dev, call, *args, workspace.data_ptr(),
                           workspace.numel() * workspace.element_size(), *sizes)
    if status == nat.ERR_WORKSPACE:
        nbytes = lib.msattn_fp4_workspace_bytes(B, q_len, H, KVH, D, max_context, code)
        with current(dev):
            workspace = _workspace(dev, nbytes)
        status = on_device(dev, call, *args, workspace.data_ptr(), nbytes, *sizes)
    if status:
        _check("msattn_paged_attention_fp4", status, k_cache, v_cache)
    return out if given is None else given.copy_(out)
