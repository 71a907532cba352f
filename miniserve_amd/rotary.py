"""miniserve_amd.rotary -- rotated queries and keys on their way into the paged cache.

``write_kv_rope`` is ``write_kv`` (miniserve/attention.py:111-133) with rotate-half RoPE
(miniserve/attention.py:41-62) of the keys on the way and of the step's queries beside them, in
one launch of libmsattn.so (msattn_write_kv_rope). The single-token form that goes on to attend is
``paged_attention_append(..., rope=)``.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Sequence

import torch

from . import _native as nat

_I64x3 = ctypes.c_int64 * 3
_SOURCES = (torch.float32, torch.float16, torch.bfloat16)


def current(dev: torch.device):
    """A context with `dev` current."""
    return contextlib.nullcontext() if dev.index is None or \
        torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def on_device(dev: torch.device, fn, *args) -> int:
    """fn(*args, stream) with `dev` current and torch's current stream on it."""
    if dev.index is None or torch._C._cuda_getDevice() == dev.index:
        return fn(*args, nat.stream_handle(dev))
    with torch.cuda.device(dev):
        return fn(*args, nat.stream_handle(dev))


def rope_table(t, dev: torch.device, what: str) -> torch.Tensor:
    """A rotation table as the kernels read it: fp32 [max_pos, dims], contiguous, on `dev`."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != dev:
        t = torch.as_tensor(t, device=dev).to(torch.float32)
    if t.ndim != 2 or t.shape[0] < 1:
        raise ValueError(f"{what} must be [max_pos, dims] with at least one position")
    return t if t.is_contiguous() else t.contiguous()


def on_16_bytes(t: torch.Tensor) -> torch.Tensor:
    """`t`, or a copy where it lies off 16 bytes (the decode kernels read 16 of a table at once)."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def extent(t: torch.Tensor) -> tuple[int, int]:
    """First byte that `t` addresses and the one past its last."""
    lo = t.data_ptr()
    if t.is_contiguous():
        return lo, lo + t.nbytes
    if t.numel() == 0:
        return lo, lo
    if t.ndim == 4:
        (a, b, c, d), (sa, sb, sc, sd) = t.shape, t.stride()
        last = (a - 1) * sa + (b - 1) * sb + (c - 1) * sc + (d - 1) * sd
    else:
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return lo, lo + (last + 1) * t.element_size()


def _rows_apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [batch, tokens, heads, dims] views of one buffer interleave token by token
    without sharing an element, as the slices of a fused projection do."""
    if a.dtype != b.dtype or a.stride()[:2] != b.stride()[:2] or a.shape[:2] != b.shape[:2]:
        return False
    token, batch, es = a.stride(1), a.stride(0), a.element_size()
    gap = b.data_ptr() - a.data_ptr()
    if gap < 0:
        return _rows_apart(b, a)
    row = [(t.shape[2] - 1) * t.stride(2) + t.shape[3] for t in (a, b)]
    return gap % es == 0 and row[0] <= gap // es and gap // es + row[1] <= token and \
        (a.shape[0] == 1 or batch >= a.shape[1] * token)


def _spans(tensors: Sequence[torch.Tensor]) -> list[tuple[int, int, torch.Tensor]]:
    return [(*extent(t), t) for t in tensors]


def _clear(t: torch.Tensor, written: Sequence[tuple[int, int, torch.Tensor]]) -> bool:
    lo, hi = extent(t)
    for wlo, whi, w in written:
        if lo < whi and wlo < hi and not (t.ndim == w.ndim == 4 and _rows_apart(t, w)):
            return False
    return True


def _apart(t: torch.Tensor, written: Sequence[torch.Tensor]) -> bool:
    return _clear(t, _spans(written))


def _source(t: torch.Tensor, written: Sequence[tuple[int, int, torch.Tensor]]) -> torch.Tensor:
    """`t` as the kernel may read it through its strides: rows of contiguous dims that share no
    memory with the `_spans` that the call writes (a copy otherwise)."""
    if t.is_neg():
        t = t.resolve_neg()
    if t.stride(3) != 1 and t.shape[3] != 1 or not _clear(t, written):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def write_kv_rope(query: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor,
                  k_cache: torch.Tensor, v_cache: torch.Tensor, block_table, start,
                  cos: torch.Tensor, sin: torch.Tensor, position=None, *,
                  out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Rotate a step's queries and keys, and scatter the keys and values into the cache.

    ``query`` [batch, tokens, heads, head_dim] (or None), ``k``/``v`` [batch, tokens, kv_heads,
    head_dim] of one fp32, fp16 or bf16 type, in any strides: the views of a fused projection are
    read where they lie. Row b's token t goes to cache position start[b] + t (``start``: an int,
    one entry per row, or an int tensor); tokens on holes of the block table or outside it are
    not written. It is rotated at that position, or at ``position``: an int, [batch] positions of
    the rows' first tokens, or [batch, tokens]. ``cos``/``sin`` [max_pos, rotary_dim] are read as
    fp32, positions clamped to [0, max_pos); the first rotary_dim dims (even) are rotated
    (x * cos + rotate_half(x) * sin), the others kept.

    Everything is computed in fp32 and rounded once: queries to their type, keys and values to
    the cache's. Returns the rotated queries, contiguous, or ``out``, which may be ``query``
    itself (rotated in place). Two tokens of one call must not land in one cache slot: parts of
    either's rows may remain there.
    """
    if not (k_cache.is_cuda and v_cache.is_cuda and k.is_cuda and v.is_cuda):
        for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("k", k), ("v", v)):
            _att._require_gpu(t, name)
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError("k and v must both be [batch, tokens, kv_heads, head_dim]")
    cache_stride = k_cache.stride()
    if k_cache.ndim != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype or \
            cache_stride != v_cache.stride():
        raise ValueError("k_cache and v_cache must share a [num_blocks, block_size, kv_heads, "
                         "head_dim] shape, dtype and strides")
    B, T, KVH, D = k.shape
    nb, bs, cache_heads, cache_dim = k_cache.shape
    if cache_heads != KVH or cache_dim != D:
        raise ValueError("k/v heads or head_dim do not match the cache")
    if cache_stride[3] != 1:
        raise ValueError("cache head_dim must be contiguous")
    if D > nat.MAX_HEAD_DIM:
        raise ValueError(f"head_dim {D}: the kernels take head sizes up to {nat.MAX_HEAD_DIM}")
    dev, dtype = k_cache.device, k.dtype
    if query is None:
        if out is not None:
            raise ValueError("out holds rotated queries: it needs a query")
    else:
        if not query.is_cuda:
            _att._require_gpu(query, "query")
        if query.ndim != 4:
            raise ValueError("query must be [batch, tokens, heads, head_dim] beside k and v")
        qB, qT, H, qD = query.shape
        if qB != B or qT != T or qD != D or H == 0:
            raise ValueError("query must be [batch, tokens, heads, head_dim] beside k and v")
        if query.dtype != dtype:
            raise ValueError("query must have k's dtype")
    if v.dtype != dtype:
        raise ValueError("v must have k's dtype")
    if dtype not in _SOURCES:
        raise ValueError(f"unsupported dtype for a rotation: {dtype}")
    if v_cache.device != dev or k.device != dev or v.device != dev or \
            query is not None and query.device != dev or out is not None and out.device != dev:
        raise ValueError("query, k, v, out and the caches must be on one device")
    cos, sin = rope_table(cos, dev, "cos"), rope_table(sin, dev, "sin")
    R = cos.shape[1]
    if cos.shape != sin.shape or R % 2 or not 0 < R <= D:
        raise ValueError(f"cos/sin must share one [max_pos, rotary_dim] shape, rotary_dim even and "
                         f"at most {D}")
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or
                            out.stride(3) != 1 or
                            any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride()))):
        raise ValueError("out must have the query's shape and dtype, rows of contiguous dims and "
                         "no element twice")
    if B == 0 or T == 0 or KVH == 0 or nb == 0:
        return None if query is None else _rest(query, out)
    table = _att.block_table_i32(block_table, dev)
    if table.shape[0] < B:
        raise ValueError("block_table has fewer rows than k")
    if table.shape[1] == 0:
        raise ValueError("block_table has no columns")
    if isinstance(start, torch.Tensor):
        start = _att.narrow_i32(start)
    starts = _att.starts_i32(start, B, dev)
    pos, per_token = None, 0
    if position is not None:
        pos = _att.narrow_i32(torch.as_tensor(position, device=dev))
        if pos.ndim == 0:
            pos = pos.expand(B)
        if tuple(pos.shape) not in ((B,), (B, T)):
            raise ValueError(f"position must be an int, [{B}] or [{B}, {T}]")
        per_token = 1 if pos.ndim == 2 else 0
        pos = pos.contiguous()
    q_args = (None, None, None, None, 0)
    written = _spans((k_cache, v_cache))
    if query is not None:
        if out is None:
            out = torch.empty((B, T, H, D), dtype=dtype, device=dev)
            q = _source(query, written)
        else:
            if not _clear(out, written):
                raise ValueError("out shares memory with a cache")
            written += _spans((out,))
            in_place = out.data_ptr() == query.data_ptr() and out.stride() == query.stride()
            q = query if in_place and not query.is_neg() else _source(query, written)
        q_args = (q.data_ptr(), _I64x3(*q.stride()[:3]), out.data_ptr(),
                  _I64x3(*out.stride()[:3]), H)
    ks, vs = _source(k, written), _source(v, written)
    status = on_device(
        dev, nat.lib().msattn_write_kv_rope, *q_args[:4], ks.data_ptr(), _I64x3(*ks.stride()[:3]),
        vs.data_ptr(), _I64x3(*vs.stride()[:3]), k_cache.data_ptr(), v_cache.data_ptr(),
        cache_stride[0], cache_stride[1], cache_stride[2], table.data_ptr(),
        starts.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        None if pos is None else pos.data_ptr(), per_token, cos.shape[0], R, B, T, q_args[4],
        KVH, D, bs, nb, table.shape[1], nat.dtype_code(dtype), nat.dtype_code(k_cache.dtype))
    nat.check("msattn_write_kv_rope", status)
    return out


def _rest(query: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    """The answer of a call without a token (or without a KV head to write): nothing to rotate."""
    if query.numel():
        raise ValueError("a query needs keys and values beside it")
    return torch.empty(query.shape, dtype=query.dtype, device=query.device) if out is None else out


from . import attention as _att  # noqa: E402  (which imports this module's names)
