"""Cases of the operators that put rotated keys into a paged cache and read prefixes once.

Three operators, each in its plain form (elementary torch operations in 32 bits) and, where
`own` is true, through the package's entry points:

  write   the rotation of a step's queries and keys, and the scatter of the rotated keys and of
          the values into the paged cache: a chunk of a prompt, or one token a sequence
  decode  one layer of a decode step: the new token's key rotated and appended with its value,
          the query rotated, attention over everything cached so far
  shared  attention for a batch whose rows come in groups, each group behind a prefix of its own
          (the same physical pages), one query token a row or a few (drafts being verified)

Lengths and group sizes belong to the case; the seed of `prepare` draws values and pages.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16,
          "fp8": torch.float8_e4m3fn}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2, "fp8": 1}
# (query heads, KV heads, head_dim) of the repository's benchmark configurations
SMALL, LLAMA, WIDE7 = (14, 2, 64), (32, 8, 128), (28, 4, 128)


def _write(heads, q, kv, batch, tokens, start, rot=None, views=True, name=None):
    c = {"op": "write", "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "q": q, "kv": kv,
         "batch": batch, "tokens": tokens, "start": start, "rot": rot or heads[2], "views": views}
    return dict(c, name=name) if name else c


def _decode(heads, q, kv, batch, lo, hi, pad=0, name=None):
    """Contexts after the append lie in [lo, hi]; the last `pad` rows are padding (no context)."""
    c = {"op": "decode", "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "q": q, "kv": kv,
         "batch": batch, "lo": lo, "hi": hi, "pad": pad}
    return dict(c, name=name) if name else c


def _shared(heads, q, kv, batch, groups, loose, tokens, prefix_lo, prefix_hi, own_lo, own_hi,
            name=None):
    """`groups` groups over the first batch - loose rows, the last `loose` rows in none; prefixes of
    prefix_lo .. prefix_hi tokens (whole pages), then own_lo .. own_hi tokens a row."""
    c = {"op": "shared", "heads": heads[0], "kv_heads": heads[1], "dim": heads[2], "q": q, "kv": kv,
         "batch": batch, "groups": groups, "loose": loose, "tokens": tokens,
         "prefix_lo": prefix_lo, "prefix_hi": prefix_hi, "own_lo": own_lo, "own_hi": own_hi}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decoded token of each of 32 sequences in a small model: launch and host latency.
        _write(SMALL, "bf16", "bf16", 32, 1, 1024, name="write_step_bf16"),
        # Two prompts' 512-token chunks, from a fused projection's views.
        _write(WIDE7, "fp16", "fp16", 2, 512, 4096, name="write_chunk_fp16"),
        # A head size off the powers of two, half of it rotated, odd lengths, in the runner's fp32.
        _write((24, 8, 96), "fp32", "fp32", 3, 1001, 77, rot=48, views=False,
               name="write_partial_fp32"),
        # Whole long prompts into an fp8 cache: the largest write.
        _write(LLAMA, "bf16", "fp8", 4, 8191, 0, name="write_prompt_fp8"),
        # Four short chats in the runner's default types: latency.
        _decode(SMALL, "fp32", "fp32", 4, 128, 512, name="decode_small_fp32"),
        # A graph bucket of a small model, three of its rows padding.
        _decode(SMALL, "bf16", "bf16", 32, 512, 2048, pad=3, name="decode_32_bf16"),
        # Few longer contexts of a 7B-class model over an fp8 cache.
        _decode(WIDE7, "fp16", "fp8", 16, 1024, 4096, name="decode_wide_fp8"),
        # The headline batch: 64 ragged sequences, bandwidth-bound; the largest read.
        _decode(LLAMA, "bf16", "bf16", 64, 1024, 8192, name="decode_64_bf16"),
        # Six chats behind two short system prompts in a small model: latency.
        _shared(SMALL, "bf16", "bf16", 6, 2, 0, 1, 256, 512, 16, 128, name="shared_small_bf16"),
        # A served batch: eight system prompts or documents, a few rows without one.
        _shared(LLAMA, "bf16", "bf16", 64, 8, 4, 1, 1024, 8192, 64, 1024,
                name="shared_groups_bf16"),
        # Four-token drafts being verified behind four prompts.
        _shared(WIDE7, "fp16", "fp16", 32, 4, 0, 4, 2048, 4096, 100, 600,
                name="shared_draft_fp16"),
        # One long system prompt under a large batch, fp8 cache.
        _shared(LLAMA, "bf16", "fp8", 128, 1, 0, 1, 8192, 8192, 256, 2048,
                name="shared_system_fp8"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm, odd ones among them."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("write", "decode", "shared"))
    heads = rng.choice((SMALL, LLAMA, WIDE7, (16, 2, 64), (8, 8, 128), (16, 4, 128), (12, 12, 64)))
    if op == "write":
        dim = rng.choice((heads[2], 64, 80, 96, 128, 256))
        q, kv = rng.choice((("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp8"), ("fp16", "fp8"),
                            ("fp32", "fp32"), ("bf16", "fp32"), ("fp32", "bf16")))
        rot = rng.choice((dim, dim, dim, dim // 2, 32))
        batch = _spread(rng, 1, 64)
        tokens = _spread(rng, 1, max(1, 24000 * 64 // (batch * dim)))
        return _write((heads[0], heads[1], dim), q, kv, batch, tokens, _spread(rng, 1, 2000), rot,
                      rng.random() < 0.6)
    q, kv = rng.choice((("bf16", "bf16"), ("fp16", "fp16"), ("bf16", "fp8"), ("fp16", "fp8"))
                       + ((("fp32", "fp32"),) if op == "decode" else ()))
    per = 2 * heads[1] * heads[2] * BYTES[kv]  # bytes a cached token
    if op == "decode":
        batch = _spread(rng, 1, 128)
        hi = _spread(rng, 128, max(129, min(16384, 700_000_000 // (per * batch))))
        return _decode(heads, q, kv, batch, max(1, hi // rng.choice((1, 2, 8))), hi,
                       rng.choice((0, 0, batch // 5)))
    batch = _spread(rng, 2, 128)
    groups = _spread(rng, 1, max(1, min(16, batch // 2)))
    tokens = rng.choice((1, 1, 1, 2, 3, 5, 8))
    prefix = _spread(rng, 64, 8192)
    most = _spread(rng, 32, 2000 if batch < 64 else 1000)
    return _shared(heads, q, kv, batch, groups, rng.choice((0, 0, batch // 8)), tokens,
                   max(PAGE, prefix // rng.choice((1, 2, 4))), prefix, max(tokens, most // 8), most)


def _rng(case):
    """Draws the lengths of a case, the same ones each time."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _shape(case):
    """(context lengths, group rows, prefix pages) of a decode or shared case."""
    rng = _rng(case)
    if case["op"] == "decode":
        lens = [_spread(rng, case["lo"], case["hi"]) for _ in range(case["batch"] - case["pad"])]
        lens[0] = case["hi"]
        return lens + [0] * case["pad"], [0], []
    n, g = case["batch"] - case["loose"], case["groups"]
    cuts = sorted(rng.sample(range(1, n), g - 1)) if g > 1 else []
    rows = [0] + cuts + [n]
    pages = [max(1, _spread(rng, case["prefix_lo"], case["prefix_hi"]) // PAGE) for _ in range(g)]
    lens = [_spread(rng, case["own_lo"], case["own_hi"]) for _ in range(case["batch"])]
    for i in range(g):
        for b in range(rows[i], rows[i + 1]):
            lens[b] += pages[i] * PAGE
    return lens, rows, pages


def _pages(case, lens, rows, pages):
    """The block table's page numbers before shuffling, -1 past a row's end, and how many there
    are: a group's rows begin with the same pages."""
    width = max(1, max(-(-n // PAGE) for n in lens))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    first = [0] * len(lens)
    for i, p in enumerate(pages):
        for b in range(rows[i], rows[i + 1]):
            table[b, :p] = torch.arange(at, at + p, dtype=torch.int32)
            first[b] = p
        at += p
    for b, n in enumerate(lens):
        w = -(-n // PAGE) - first[b]
        if w > 0:
            table[b, first[b]:first[b] + w] = torch.arange(at, at + w, dtype=torch.int32)
            at += w
    return table, max(1, at)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    B, q, kv = case["batch"], DTYPES[case["q"]], DTYPES[case["kv"]]
    T = case.get("tokens", 1)
    if case["op"] == "write":
        lens, rows, pages = [case["start"] + T] * B, [0], []
    else:
        lens, rows, pages = _shape(case)
    table, n = _pages(case, lens, rows, pages)
    table = table.to(dev)
    shuffle = torch.randperm(n, generator=g, device=dev).to(torch.int32)
    table = torch.where(table >= 0, shuffle[table.clamp(min=0).long()], table).contiguous()

    def values(*shape, dtype=q):
        return torch.randn(*shape, generator=g, device=dev).to(dtype)

    s = {"op": case["op"], "table": table, "k_cache": values(n, PAGE, KVH, D, dtype=kv),
         "v_cache": values(n, PAGE, KVH, D, dtype=kv), "max_context": max(lens),
         "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if case["op"] == "shared":
        s["q"] = values(B, T, H, D)
        s["group_rows"] = torch.tensor(rows, dtype=torch.int32, device=dev)
        s["prefix_pages"] = torch.tensor(pages, dtype=torch.int32, device=dev)
        return s
    if case["op"] == "write" and case["views"]:  # a fused projection's output, as views
        qkv = values(B, T, H + 2 * KVH, D)
        s["q"], s["k"], s["v"] = qkv[:, :, :H], qkv[:, :, H:H + KVH], qkv[:, :, H + KVH:]
    else:
        s["q"], s["k"], s["v"] = values(B, T, H, D), values(B, T, KVH, D), values(B, T, KVH, D)
    # rotation tables as a model keeps them: fp32, angles taken in 64 bits
    rot = case.get("rot", D)
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    angle = torch.arange(max(lens), device=dev, dtype=torch.float64)[:, None] * inv[None, :]
    s["cos"] = torch.cat((angle.cos(), angle.cos()), dim=1).float()
    s["sin"] = torch.cat((angle.sin(), angle.sin()), dim=1).float()
    s["start"] = s["lens"] - T
    return s


def _rotate(x, cos, sin):
    """Rotate-half of the first cos.shape[-1] dims, in 32 bits."""
    r = cos.shape[-1]
    a = x[..., :r]
    turned = torch.cat((-a[..., r // 2:], a[..., :r // 2]), dim=-1)
    return torch.cat((a * cos + turned * sin, x[..., r:]), dim=-1)


def _bits(cache):
    return cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache


def _append(s, k, v):
    """k, v [batch, tokens, heads, dim] in 32 bits to the positions start + t of the cache."""
    B, T = k.shape[:2]
    pos = s["start"][:, None].long() + torch.arange(T, device=k.device)
    page = torch.gather(s["table"].long(), 1, pos.clamp(min=0) // PAGE)
    live = (pos >= 0) & (page >= 0)
    slot = (page[live], (pos % PAGE)[live])
    for cache, x in ((s["k_cache"], k), (s["v_cache"], v)):
        _bits(cache)[slot] = _bits(x.to(cache.dtype)[live])


def _attend(s, q):
    """Causal attention of q [batch, tokens, heads, dim] (32 bits) over each row's context."""
    B, T, H, D = q.shape
    KVH = s["k_cache"].shape[2]
    at = s["table"].clamp(min=0).long()

    def gather(cache):
        x = _bits(cache)[at]
        return x.view(cache.dtype).float().reshape(B, -1, KVH, D).transpose(1, 2)

    k = gather(s["k_cache"])
    rows = q.reshape(B, T, KVH, H // KVH, D).transpose(1, 2).reshape(B, KVH, -1, D)
    scores = torch.matmul(rows, k.transpose(2, 3).contiguous()) / math.sqrt(D)
    del k
    key = torch.arange(scores.shape[3], device=q.device)
    last = s["lens"][:, None].long() - T + torch.arange(T, device=q.device)  # [batch, tokens]
    seen = key <= last[:, :, None]
    seen = seen[:, None, :, None].expand(B, KVH, T, H // KVH, -1).reshape(scores.shape)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(dim=3, keepdim=True)
    w = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = w.sum(dim=3, keepdim=True)
    out = torch.matmul(w, gather(s["v_cache"]).contiguous()) / torch.where(total > 0, total, 1.0)
    return out.reshape(B, KVH, T, H // KVH, D).transpose(1, 2).reshape(B, T, H, D)


def run(s):
    if own:
        from miniserve_amd import (paged_attention_append, paged_attention_shared, write_kv_rope)
        if s["op"] == "write":
            q = write_kv_rope(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"],
                              s["start"], s["cos"], s["sin"])
            return [q, s["k_cache"], s["v_cache"]]
        if s["op"] == "decode":
            out = paged_attention_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"],
                                         s["table"], s["lens"], max_context=s["max_context"],
                                         rope=(s["cos"], s["sin"]))
            return [out, s["k_cache"], s["v_cache"]]
        return [paged_attention_shared(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                       s["group_rows"], s["prefix_pages"],
                                       max_context=s["max_context"])]
    if s["op"] == "shared":
        return [_attend(s, s["q"].float()).to(s["q"].dtype)]
    pos = (s["start"][:, None].long() + torch.arange(s["q"].shape[1], device=s["q"].device))
    at = pos.clamp(min=0)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    q = _rotate(s["q"].float(), cos, sin)
    _append(s, _rotate(s["k"].float(), cos, sin), s["v"].float())
    if s["op"] == "decode":
        q = _attend(s, q)
    return [q.to(s["q"].dtype), s["k_cache"], s["v_cache"]]


def work(case):
    H, KVH, D, B = case["heads"], case["kv_heads"], case["dim"], case["batch"]
    qb, kb = BYTES[case["q"]], BYTES[case["kv"]]
    T = case.get("tokens", 1)
    if case["op"] == "write":
        rows = B * T
        tables = 2 * 4 * case["rot"] * T  # the rows' positions are the same ones
        return {"bytes": rows * D * (2 * H * qb + 2 * KVH * (qb + kb)) + tables,
                "flops": 3 * rows * case["rot"] * (H + KVH)}
    lens, rows, pages = _shape(case)
    prefix = [0] * B
    for i, p in enumerate(pages):
        for b in range(rows[i], rows[i + 1]):
            prefix[b] = p * PAGE
    cached = sum(n - p for n, p in zip(lens, prefix)) + PAGE * sum(pages)
    pairs = sum(max(0, n - T + 1 + t) for n in lens for t in range(T))
    moved = cached * 2 * KVH * D * kb + 2 * B * T * H * D * qb + 4 * (cached // PAGE) + 4 * B
    if case["op"] == "decode":  # the new rows are read in the query's type and written
        moved += 2 * B * KVH * D * qb + 2 * 4 * D * B
    return {"bytes": moved, "flops": 4 * pairs * H * D}


def exact(case, seed):
    """The definition in 64 bits, a row of the batch at a time."""
    s = prepare(case, seed)
    f64 = torch.float64
    T, D = case.get("tokens", 1), case["dim"]
    kc, vc = (_bits(s[n]).clone().view(s[n].dtype) for n in ("k_cache", "v_cache"))
    table, lens = s["table"].tolist(), s["lens"].tolist()
    q = s["q"].to(f64)
    out = []
    if case["op"] != "shared":
        half = case.get("rot", D) // 2

        def turn(x, b):  # x [tokens, heads, dim]
            y = x.clone()
            p = [max(0, lens[b] - T + t) for t in range(T)]
            c, n = s["cos"][p].to(f64)[:, None], s["sin"][p].to(f64)[:, None]
            lo, hi = x[..., :half], x[..., half:2 * half]
            y[..., :half] = lo * c[..., :half] - hi * n[..., :half]
            y[..., half:2 * half] = hi * c[..., half:] + lo * n[..., half:]
            return y

        k64, v64 = kc.to(f64), vc.to(f64)
        q = torch.stack([turn(q[b], b) for b in range(case["batch"])])
        for b in range(case["batch"]):
            new_k, new_v = turn(s["k"][b].to(f64), b), s["v"][b].to(f64)
            where = [(t, lens[b] - T + t) for t in range(T) if lens[b] - T + t >= 0]
            at = [(t, table[b][p // PAGE], p % PAGE) for t, p in where if table[b][p // PAGE] >= 0]
            if not at:
                continue
            t, page, slot = (torch.tensor(x, device=q.device) for x in zip(*at))
            k64[page, slot], v64[page, slot] = new_k[t], new_v[t]
        if case["op"] == "write":
            return [q, k64, v64]
        # the cache holds its own type: attention reads what was stored
        kc, vc = k64.to(kc.dtype), v64.to(vc.dtype)
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(lens):
        o = torch.zeros(T, case["heads"], D, dtype=f64, device=q.device)
        if n > 0:
            at = torch.tensor(table[b][:-(-n // PAGE)], device=q.device)
            k, v = (_bits(x)[at].view(x.dtype).reshape(-1, *x.shape[2:])[:n].to(f64)
                    .repeat_interleave(group, dim=1).transpose(0, 1) for x in (kc, vc))
            x = (q[b].transpose(0, 1) @ k.transpose(1, 2).contiguous()) * D ** -0.5
            later = torch.arange(n, device=q.device)[None, :] > \
                torch.arange(n - T, n, device=q.device)[:, None]
            p = torch.softmax(x.masked_fill(later, -math.inf), dim=2)
            o = torch.nan_to_num(p @ v.contiguous(), nan=0.0).transpose(0, 1)
        out.append(o)
    out = torch.stack(out)
    return [out] if case["op"] == "shared" else [out, k64, v64]
