"""miniserve_amd.shared -- attention for a batch behind several shared prefixes.

When the radix cache (miniserve/prefix_cache.py:66-96) hands several requests of a batch the same
leading pages, and other requests other ones, each group's prefix is read once for the group
(msattn_paged_attention_shared). One prefix under a whole decode batch is also
``paged_attention(..., prefix_pages=)``.
"""
from __future__ import annotations

import math

import torch

from . import _native as nat
from .attention import (_host_ints_to_device, _require_gpu, _workspace, block_table_i32,
                        context_lens_i32, narrow_i32, paged_attention)
from .rotary import current, extent, on_device


def check_groups(group_rows, prefix_pages, batch: int, width: int, dev: torch.device) -> list:
    """[group_rows, prefix_pages], host values checked and as lists, tensors on `dev` as they are (the
    host does not read them); as many of the one as the other needs."""
    out = []
    for name, x, most in (("group_rows", group_rows, batch), ("prefix_pages", prefix_pages, width)):
        if isinstance(x, torch.Tensor) and (x.dtype.is_floating_point or x.dtype.is_complex or
                                            x.dtype == torch.bool):
            raise ValueError(f"{name} must hold whole numbers")
        if isinstance(x, torch.Tensor) and x.device == dev:
            out.append(x if x.ndim == 1 else x.reshape(-1))
            continue
        given = x.reshape(-1).tolist() if isinstance(x, torch.Tensor) else list(x)
        values = [int(v) for v in given]
        if values != given:
            raise ValueError(f"{name} must hold whole numbers")
        if name == "group_rows":
            if any(a > b for a, b in zip(values, values[1:])) or \
                    any(not 0 <= v <= batch for v in values):
                raise ValueError(f"group_rows must ascend within [0, {batch}]")
        elif any(not 0 <= v <= width for v in values):
            raise ValueError(f"prefix_pages must lie within [0, {width}]")
        out.append(values)
    rows, pages = map(len, out)
    if rows != pages + 1 and not (rows == 0 and pages == 0):
        raise ValueError(f"{pages} groups need {pages + 1} group_rows, not {rows}")
    return out


def _groups_i32(group_rows, prefix_pages, batch: int, width: int, dev: torch.device
                ) -> tuple[torch.Tensor, torch.Tensor]:
    """(int32 [groups + 1], int32 [groups]) on `dev`; host values are checked."""
    rows, pages = (
        narrow_i32(x, 0, most).contiguous() if isinstance(x, torch.Tensor) else
        _host_ints_to_device(x, dev)
        for x, most in zip(check_groups(group_rows, prefix_pages, batch, width, dev), (batch, width)))
    return rows, pages


def paged_attention_shared(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           block_table, context_lens, group_rows, prefix_pages, *,
                           scale: float | None = None, max_context: int | None = None,
                           workspace: torch.Tensor | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal paged attention of ``query`` [batch, q_len, heads, head_dim] whose rows come in
    groups: rows ``group_rows[g]`` .. ``group_rows[g + 1] - 1`` hold the same physical pages in
    their first ``prefix_pages[g]`` block-table entries, and those pages are read once for the
    group. Rows in no group (before the first, after the last) share nothing.

    ``group_rows`` [groups + 1] and ``prefix_pages`` [groups] are lists (checked) or int tensors;
    on the device they are not read by the host, so the call is safe to capture, and what a graph
    reads may change between replays (values out of range are taken as the nearest bound). That a
    group's rows really share the pages is the caller's word. ``context_lens``, ``max_context``,
    ``workspace`` (zeros when first used) and ``out`` as in ``paged_attention``, whose result this
    is within float rounding, for one query token a row or several.
    """
    _require_gpu(query, "query")
    _require_gpu(k_cache, "k_cache")
    _require_gpu(v_cache, "v_cache")
    if query.ndim != 4 or k_cache.ndim != 4:
        raise ValueError("query must be [batch, q_len, heads, head_dim] and the caches "
                         "[num_blocks, block_size, kv_heads, head_dim]")
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype or \
            k_cache.stride() != v_cache.stride():
        raise ValueError("k_cache and v_cache must share shape, dtype and strides")
    B, q_len, H, D = query.shape
    nb, bs, KVH, Dk = k_cache.shape
    if Dk != D:
        raise ValueError(f"head_dim mismatch: query {D}, cache {Dk}")
    if D > nat.MAX_HEAD_DIM or D % 2:
        raise ValueError(f"head_dim {D}: the kernels take even head sizes up to "
                         f"{nat.MAX_HEAD_DIM}")
    if KVH == 0 or H % KVH:
        raise ValueError("num_heads must be a multiple of num_kv_heads")
    if k_cache.stride(3) != 1:
        raise ValueError("cache head_dim must be contiguous")
    dev = query.device
    if k_cache.device != dev or v_cache.device != dev:
        raise ValueError("query and the caches must be on one device")
    table = block_table_i32(block_table, dev)
    if table.shape[0] != B:
        raise ValueError(f"block_table has {table.shape[0]} rows for a batch of {B}")
    W = table.shape[1]
    rows, pages = _groups_i32(group_rows, prefix_pages, B, W, dev)
    groups = pages.numel()
    if groups == 0 or B == 0 or q_len == 0:
        with current(dev):
            return paged_attention(query, k_cache, v_cache, table, context_lens, scale=scale,
                                   max_context=max_context, workspace=workspace, out=out)
    lens, host_max = context_lens_i32(context_lens, dev, B)
    cap = W * bs
    if max_context is None:
        max_context = cap if host_max is None else host_max
    if host_max is not None and host_max > cap:
        raise ValueError(f"context length {host_max} exceeds the block table capacity {cap}")
    max_context = max(0, min(int(max_context), cap))
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    fresh = out is None
    if fresh:
        out = torch.empty((B, q_len, H, D), dtype=query.dtype, device=dev)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != dev or \
            not out.is_contiguous():
        raise ValueError("out must be contiguous, of the query's shape, dtype and device")
    if workspace is not None and (workspace.device != dev or not workspace.is_contiguous()):
        raise ValueError("workspace must be contiguous and on the query's device")
    lib = nat.lib()
    ws_bytes = lib.msattn_shared_workspace_bytes(B, q_len, H, KVH, D, max_context, groups)
    if ws_bytes == 0:
        raise ValueError("unsupported attention geometry")
    if workspace is None or workspace.numel() * workspace.element_size() < ws_bytes:
        workspace = _workspace(dev, ws_bytes)
    q = query.contiguous()
    if q is query and not fresh:  # a kernel reads all of it while the output is written
        (lo, hi), (olo, ohi) = extent(q), extent(out)
        if lo < ohi and olo < hi:
            q = q.clone()
    status = on_device(
        dev, lib.msattn_paged_attention_shared, q.data_ptr(), k_cache.data_ptr(),
        v_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
        table.data_ptr(), lens.data_ptr(), rows.data_ptr(), pages.data_ptr(), groups,
        out.data_ptr(), workspace.data_ptr(), ws_bytes, B, q_len, H, KVH, D, bs, nb, W,
        max_context, float(scale), nat.dtype_code(query.dtype), nat.dtype_code(k_cache.dtype))
    nat.check("msattn_paged_attention_shared", status)
    return out
