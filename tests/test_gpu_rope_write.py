"""The rotated cache write (write_kv_rope) and its single-token form (paged_attention_append with
rope) on the GPU: against the rotation in 64 bits, against each other, captured and replayed.

Tolerances. The kernels rotate in fp32: y = fl(fl(a c) + fl(b s)), so |error| <= 2^-24 (|a c| +
|b s|) from the products and 2^-24 |y| (1 + 2^-23) from the sum, together at most 2^-22 (|a c| +
|b s|); the rounding to the stored type adds half a step of it: eps / 2 |y|, or half the type's
smallest subnormal below its normal range. Unrotated elements and values are one rounding each,
which torch makes too: they are equal bit for bit.
"""
import math

import pytest
import torch

from miniserve_amd import (PagedAttention, _native as nat, kernel_route, paged_attention,
                           paged_attention_append, write_kv_rope)
from miniserve_amd.graphs import DecodeLayer, GraphedDecodeRunner
from oracle import dense

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
SUBNORMAL = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133, FP8: 2.0 ** -9}


def note(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


def tables(max_pos, R, device, dtype=F32, base=10000.0):
    """Tables whose two halves differ, as the formula allows."""
    inv = base ** (-torch.arange(R, dtype=torch.float64) / R)
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * inv
    return a.cos().to(dtype).to(device), a.sin().to(dtype).to(device)


def rotate64(x, cos, sin, pos):
    """(rotated, |a c| + |b s|) of x [B, T, heads, D] in 64 bits at pos [B, T] (CPU)."""
    x, R = x.double().cpu(), cos.shape[1]
    p = pos.clamp(0, cos.shape[0] - 1)
    c, s = cos.double().cpu()[p][:, :, None], sin.double().cpu()[p][:, :, None]
    a = x[..., :R]
    turned = torch.cat((-a[..., R // 2:], a[..., :R // 2]), dim=-1)
    y, size = x.clone(), torch.zeros_like(x)
    y[..., :R] = a * c + turned * s
    size[..., :R] = (a * c).abs() + (turned * s).abs()
    return y, size


def check_rounded(got, want, size, dtype, what):
    err = (got.cpu().double() - want).abs()
    half = torch.finfo(dtype).eps / 2
    bound = half * want.abs() * (1 + half) + SUBNORMAL[dtype] / 2 + 2.0 ** -22 * size
    worst = (err - bound).max().item()
    assert worst <= 0, f"{what}: {worst:.3e} over the bound"


def bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def check_write(q, k, v, kc0, vc0, kc, vc, out, table, start, cos, sin, pos=None, holes=True):
    """A call's outputs against 64 bits; everything else in the caches as it was."""
    B, T = k.shape[:2]
    bs, W, nb = kc.shape[1], table.shape[1], kc.shape[0]
    at = torch.tensor(start)[:, None] + torch.arange(T)
    pos = at if pos is None else pos
    if q is not None:
        y, size = rotate64(q, cos, sin, pos)
        check_rounded(out, y, size, q.dtype, "query")
    y, size = rotate64(k, cos, sin, pos)
    want_k, want_v = bits(kc0).cpu().clone(), bits(vc0).cpu().clone()
    got_k, got_v = kc.cpu(), vc.cpu()
    vals = bits(v.cpu().contiguous().to(kc.dtype))
    R, tab = cos.shape[1], table.cpu().tolist()
    for b in range(B):
        for t in range(T):
            p = int(at[b, t])
            page = tab[b][p // bs] if 0 <= p < W * bs else -1
            if not 0 <= page < nb:
                continue
            s = p % bs
            row = got_k[page, s]
            check_rounded(row, y[b, t], size[b, t], kc.dtype, f"key {b},{t}")
            same = bits(k[b, t, :, R:].cpu().contiguous().to(kc.dtype))
            assert torch.equal(bits(row)[:, R:], same), "dims past the rotation"
            want_k[page, s] = bits(row)  # checked: now everything else
            want_v[page, s] = vals[b, t]
    assert torch.equal(bits(got_k), want_k) and torch.equal(bits(got_v), want_v)


# name -> (H, KVH, D, R, source, cache, B, T, block size, layout)
WRITES = {
    "one token, one head": (1, 1, 64, 64, BF16, BF16, 1, 1, 16, "dense"),
    "decode step of a small model": (14, 2, 64, 64, F32, F32, 5, 1, 16, "dense"),
    "fused views bf16": (28, 4, 128, 128, BF16, BF16, 2, 37, 16, "fused"),
    "fp8 cache": (8, 8, 128, 128, F16, FP8, 3, 21, 16, "fused"),
    "fp8 cache from fp32": (4, 2, 64, 64, F32, FP8, 2, 19, 16, "dense"),
    "fp32 cache from bf16": (4, 4, 128, 128, BF16, F32, 2, 18, 32, "heads first"),
    "bf16 cache from fp32": (6, 3, 96, 96, F32, BF16, 2, 17, 16, "dense"),
    "fp16 cache from bf16": (6, 3, 80, 80, BF16, F16, 2, 17, 48, "dense"),
    "half the dims": (8, 2, 96, 48, BF16, BF16, 2, 33, 16, "dense"),
    "a quarter, odd chunks": (4, 2, 80, 16, F16, F16, 2, 9, 16, "dense"),
    "two dims rotated": (4, 2, 64, 2, BF16, BF16, 2, 5, 16, "dense"),
    "head_dim 256": (4, 1, 256, 256, BF16, BF16, 2, 6, 16, "fused"),
    "head_dim 6": (3, 3, 6, 6, F16, F16, 2, 7, 5, "dense"),
    "head_dim 2 from fp32": (2, 1, 2, 2, F32, F32, 3, 4, 1, "dense"),
    "odd base": (4, 2, 64, 64, BF16, BF16, 2, 11, 16, "off by one"),
    "pages of 24": (4, 2, 64, 64, BF16, BF16, 2, 50, 24, "dense"),
    "padded pool": (4, 2, 64, 64, BF16, BF16, 2, 20, 16, "padded pool"),
    "many tokens": (8, 2, 64, 64, BF16, BF16, 1, 700, 16, "fused"),
}


def sources(H, KVH, D, dtype, B, T, layout, g, device):
    def rnd(*s):
        return (torch.randn(*s, generator=g) * 3).to(dtype).to(device)
    if layout == "fused":
        x = rnd(B, T, H + 2 * KVH, D)
        return x[:, :, :H], x[:, :, H:H + KVH], x[:, :, H + KVH:]
    if layout == "heads first":
        return tuple(rnd(B, n, T, D).transpose(1, 2) for n in (H, KVH, KVH))
    if layout == "off by one":
        return tuple(rnd(B * T * n * D + 1)[1:].view(B, T, n, D) for n in (H, KVH, KVH))
    return rnd(B, T, H, D), rnd(B, T, KVH, D), rnd(B, T, KVH, D)


def pool(nb, bs, KVH, D, dtype, g, device, layout="dense"):
    extra = 3 if layout == "padded pool" else 0
    def one():
        x = torch.randn(nb, bs, KVH, D + extra, generator=g).to(dtype).to(device)
        return x[..., :D]
    return one(), one()


@pytest.mark.parametrize("name", list(WRITES))
def test_write_against_64_bits(device, name):
    H, KVH, D, R, st, kt, B, T, bs, layout = WRITES[name]
    g = torch.Generator().manual_seed(H * 1000 + D + T)
    q, k, v = sources(H, KVH, D, st, B, T, layout, g, device)
    W = -(-(T + 40) // bs)
    nb = B * W + 3
    kc, vc = pool(nb, bs, KVH, D, kt, g, device, layout)
    kc0, vc0 = kc.clone(), vc.clone()
    table = torch.randperm(nb, generator=g)[:B * W].view(B, W).to(torch.int32)
    start = [int(x) for x in torch.randint(0, 40, (B,), generator=g)]
    cos, sin = tables(T + 60, R, device)
    note(f"write {name}")
    out = write_kv_rope(q, k, v, kc, vc, table.to(device), start, cos, sin)
    assert out.is_contiguous() and out.shape == q.shape and out.dtype == q.dtype
    check_write(q, k, v, kc0, vc0, kc, vc, out, table, start, cos, sin)


@pytest.mark.parametrize("D", [64, 6])
def test_holes_ends_and_starts_outside(device, D):
    """Holes, page ids past the pool, positions before the table and past its end, and a start
    near the largest int: those tokens are rotated, not written."""
    g = torch.Generator().manual_seed(D)
    B, T, H, KVH, bs, W, nb = 6, 40, 3, 1, 16, 3, 20
    q, k, v = sources(H, KVH, D, BF16, B, T, "dense", g, device)
    kc, vc = pool(nb, bs, KVH, D, BF16, g, device)
    kc0, vc0 = kc.clone(), vc.clone()
    table = torch.randperm(nb, generator=g)[:B * W].view(B, W).to(torch.int32)
    table[0, 1], table[1, 0], table[1, 2] = -1, nb, 2 ** 31 - 1
    start = [0, 3, -7, 30, W * bs, 2 ** 31 - 5]
    cos, sin = tables(64, D, device)
    note(f"holes head_dim {D}")
    out = write_kv_rope(q, k, v, kc, vc, table.to(device), start, cos, sin)
    check_write(q, k, v, kc0, vc0, kc, vc, out, table, start, cos, sin)


@pytest.mark.parametrize("form", ["rows", "tokens", "int", "outside"])
def test_positions_of_their_own(device, form):
    g = torch.Generator().manual_seed(5)
    B, T, H, KVH, D, bs, W = 3, 18, 4, 2, 64, 16, 2
    q, k, v = sources(H, KVH, D, F16, B, T, "fused", g, device)
    kc, vc = pool(B * W, bs, KVH, D, F16, g, device)
    kc0, vc0 = kc.clone(), vc.clone()
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32)
    cos, sin = tables(50, D, device)
    given, full = {
        "rows": (torch.tensor([7, 0, 30]), torch.tensor([7, 0, 30])[:, None] + torch.arange(T)),
        "tokens": (lambda p: (p, p))(torch.randint(0, 50, (B, T), generator=g)),
        "int": (9, (9 + torch.arange(T)).expand(B, T)),
        "outside": (torch.tensor([45, -20, 2 ** 31 - 3]),
                    torch.tensor([45, -20, 2 ** 31 - 3])[:, None] + torch.arange(T)),
    }[form]
    note(f"positions {form}")
    out = write_kv_rope(q, k, v, kc, vc, table.to(device), [2, 0, 5], cos, sin, given)
    check_write(q, k, v, kc0, vc0, kc, vc, out, table, [2, 0, 5], cos, sin, full)


def test_in_place_and_without_a_query(device):
    g = torch.Generator().manual_seed(6)
    B, T, H, KVH, D, bs, W = 2, 33, 4, 2, 64, 16, 4
    for dtype, layout in ((BF16, "fused"), (F32, "dense")):
        q, k, v = sources(H, KVH, D, dtype, B, T, layout, g, device)
        table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32).to(device)
        cos, sin = tables(64, D, device)
        kc, vc = pool(B * W, bs, KVH, D, dtype, g, device)
        a, b, c = (kc.clone(), vc.clone()), (kc.clone(), vc.clone()), (kc, vc)
        note(f"in place {dtype}")
        want = write_kv_rope(q, k, v, *a, table, 3, cos, sin)
        assert write_kv_rope(None, k, v, *b, table, 3, cos, sin) is None
        k0 = k.clone()
        got = write_kv_rope(q, k, v, *c, table, 3, cos, sin, out=q)
        assert got is q and torch.equal(q, want) and torch.equal(k, k0)
        for x in (b, c):
            assert torch.equal(x[0], a[0]) and torch.equal(x[1], a[1])


def test_sources_that_share_memory_with_what_is_written(device):
    """Keys that lie in the cache, a query that overlaps out a token later: copied first."""
    g = torch.Generator().manual_seed(7)
    B, T, H, KVH, D, bs = 1, 16, 2, 2, 64, 16
    kc, vc = pool(4, bs, KVH, D, BF16, g, device)
    k, v = kc[1:2], kc[2:3]
    q_buf = torch.randn(1, T + 1, H, D, generator=g).to(BF16).to(device)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device=device)
    cos, sin = tables(64, D, device)
    a = (kc.clone(), vc.clone())
    note("shared memory")
    want = write_kv_rope(q_buf[:, :-1].clone(), k.clone(), v.clone(), *a, table, 8, cos, sin)
    got = write_kv_rope(q_buf[:, :-1], k, v, kc, vc, table, 8, cos, sin, out=q_buf[:, 1:])
    assert torch.equal(got, want) and torch.equal(kc, a[0]) and torch.equal(vc, a[1])
    with pytest.raises(ValueError, match="shares memory"):
        write_kv_rope(want, k, v, kc, vc, table, 8, cos, sin, out=kc[0:1])


def test_refusals(device):
    g = torch.Generator().manual_seed(8)
    q, k, v = sources(4, 2, 64, BF16, 2, 3, "dense", g, device)
    kc, vc = pool(8, 16, 2, 64, BF16, g, device)
    cos, sin = tables(16, 64, device)
    table = torch.arange(8, dtype=torch.int32, device=device).view(2, 4)
    def call(q=q, k=k, v=v, kc=kc, vc=vc, table=table, start=0, cos=cos, sin=sin, **kw):
        write_kv_rope(q, k, v, kc, vc, table, start, cos, sin, **kw)
    for bad in (dict(k=k[:1]), dict(v=v[:, :1]), dict(q=q[:1]), dict(q=q[..., :32]),
                dict(q=q.float()), dict(v=v.half()), dict(k=k.to(FP8), v=v.to(FP8), q=None),
                dict(cos=cos[:, :32]), dict(cos=cos[:, :63], sin=sin[:, :63]),
                dict(cos=cos.repeat(1, 2), sin=sin.repeat(1, 2)), dict(cos=cos[0]),
                dict(cos=cos[:0], sin=sin[:0]), dict(vc=vc[:4]), dict(vc=vc.half()),
                dict(table=table[:1]), dict(start=[0]), dict(position=[1, 2, 3]),
                dict(out=q[:1]), dict(out=q.float()), dict(q=None, out=q),
                dict(out=q[:, :1].expand(2, 3, 4, 64)), dict(kc=kc[..., :32], vc=vc[..., :32]),
                dict(kc=kc.transpose(2, 3), vc=vc.transpose(2, 3)),
                dict(table=table[:, :0])):
        with pytest.raises(ValueError):
            call(**bad)
    empty = write_kv_rope(q[:, :0], k[:, :0], v[:, :0], kc, vc, table, 0, cos, sin)
    assert empty.shape == (2, 0, 4, 64)


def test_offsets_past_32_bits(device):
    """Pages whose elements lie past 2^31 in an fp8 pool, and long strides in the sources."""
    KVH, D, bs = 8, 128, 16
    nb = (2 ** 31) // (bs * KVH * D) + 9
    kc = torch.zeros(nb, bs, KVH, D, dtype=torch.uint8, device=device).view(FP8)
    vc = torch.zeros(nb, bs, KVH, D, dtype=torch.uint8, device=device).view(FP8)
    g = torch.Generator().manual_seed(9)
    T = 20
    k, v = (torch.randn(1, T, KVH, D, generator=g).to(BF16).to(device) for _ in range(2))
    table = torch.tensor([[nb - 1, nb - 8]], dtype=torch.int32)
    cos, sin = tables(32, D, device)
    note("offsets past 32 bits")
    write_kv_rope(None, k, v, kc, vc, table.to(device), 4, cos, sin)
    tail = nb - 9
    small = torch.tensor([[8, 1]], dtype=torch.int32)
    zero = torch.zeros(9, bs, KVH, D, dtype=torch.uint8).view(FP8)
    check_write(None, k, v, zero, zero, kc[tail:], vc[tail:], None, small, [4], cos, sin)
    assert not bits(kc)[:tail].any() and not bits(vc)[:tail].any()


def test_another_stream_and_capture(device):
    """On a side stream, and captured: three replays on new values and starts, eager work between."""
    g = torch.Generator().manual_seed(10)
    B, T, H, KVH, D, bs, W = 4, 1, 14, 2, 64, 16, 8
    q, k, v = sources(H, KVH, D, BF16, B, T, "dense", g, device)
    kc, vc = pool(B * W, bs, KVH, D, FP8, g, device)
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32).to(device)
    start = torch.zeros(B, dtype=torch.int32, device=device)
    cos, sin = tables(W * bs, D, device)
    out = torch.empty_like(q)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        write_kv_rope(q, k, v, kc, vc, table, start, cos, sin, out=out)
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write_kv_rope(q, k, v, kc, vc, table, start, cos, sin, out=out)
    for step in range(3):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        start.copy_(torch.randint(0, W * bs, (B,), generator=g))
        a = (kc.clone(), vc.clone())
        note(f"replay {step}")
        graph.replay()
        want = write_kv_rope(q, k, v, *a, table, start, cos, sin)
        assert torch.equal(out, want)
        assert torch.equal(bits(kc), bits(a[0])) and torch.equal(bits(vc), bits(a[1]))


# ------------------------------------------------------------------ the single-token form

# name -> (H, KVH, D, query, cache, batch, table pages, window, expected route)
APPENDS = {
    "C2 geometry bf16": (14, 2, 64, BF16, BF16, 32, 64, 0, "partition-fused"),
    "C5 geometry bf16, wide shape": (28, 4, 128, BF16, BF16, 16, 288, 0, "partition-fused"),
    "one query head a KV head": (4, 4, 128, F16, F16, 8, 32, 0, "partition-fused"),
    "two query heads a KV head": (4, 2, 64, F16, F16, 8, 32, 0, "partition-fused"),
    "fp16 G4 D128 window": (32, 8, 128, F16, F16, 8, 64, 300, "partition-fused"),
    "bf16 over fp8 D128": (28, 4, 128, BF16, FP8, 8, 96, 0, "partition-fused"),
    "fp16 over fp8 D64": (16, 2, 64, F16, FP8, 8, 64, 0, "partition-fused"),
    "bf16 over fp32": (14, 2, 64, BF16, F32, 16, 64, 0, "partition-fused"),
    "fp32": (14, 2, 64, F32, F32, 8, 64, 0, "partition-fused"),
    "fp32 over fp8": (14, 2, 64, F32, FP8, 8, 64, 0, "partition-fused"),
    "fp32 over bf16, D128": (8, 2, 128, F32, BF16, 8, 64, 0, "partition-fused"),
    "fp32, one query head, D128": (4, 4, 128, F32, F32, 8, 40, 0, "partition-fused"),
    "fp32, one query head, D128 (two launches)": (8, 8, 128, F32, F32, 8, 64, 0, "partition-fused"),
    "fp32 over fp16 window": (8, 1, 64, F32, F16, 8, 64, 200, "partition-fused"),
    "fp32, G16 (two launches)": (32, 2, 128, F32, F32, 8, 64, 0, "partition-fused"),
    "fp32, stream-K (two launches)": (32, 8, 128, F32, F32, 16, 512, 0, "stream-K"),
    "G16 (two launches)": (32, 2, 128, BF16, BF16, 8, 64, 0, "partition-fused"),
    "stream-K": (32, 8, 128, BF16, BF16, 16, 512, 0, "stream-K"),
    "stream-K, fp8 (two launches)": (32, 8, 128, BF16, FP8, 16, 512, 0, "stream-K"),
    "stream-K, bf16 over fp32": (32, 8, 128, BF16, F32, 16, 512, 0, "stream-K"),
    "stream-K, D64": (16, 16, 64, F16, F16, 32, 256, 0, "stream-K"),
    "head_dim 80 (two launches)": (8, 2, 80, BF16, BF16, 8, 64, 0, "generic"),
    "fp16 over bf16 (two launches)": (8, 2, 64, F16, BF16, 8, 32, 0, "generic"),
}


def append_case(name, device, seed=0):
    H, KVH, D, qt, kt, B, W, window, route = APPENDS[name]
    g = torch.Generator().manual_seed(seed + W + H + D)
    gd = torch.Generator(device=device).manual_seed(seed + W + H + D)
    nb = B * W + 8
    kc, vc = (torch.randn(nb, 16, KVH, D, generator=gd, device=device).to(kt) for _ in range(2))
    table = torch.randperm(nb, generator=g)[:B * W].view(B, W).to(torch.int32)
    lens = [int(x) for x in torch.randint(1, W * 16 + 1, (B,), generator=g)]
    lens[0], lens[1], lens[2] = 0, 1, W * 16  # a pad row, the new token alone, a full table
    if B > 3:
        table[3, (lens[3] - 1) // 16] = -1  # the new token falls on a hole
    rnd = lambda n: torch.randn(B, 1, n, D, generator=gd, device=device).to(qt)  # noqa: E731
    cos, sin = tables(W * 16, D, device)
    return (rnd(H), rnd(KVH), rnd(KVH), kc, vc, table.to(device),
            torch.tensor(lens, dtype=torch.int32, device=device), cos, sin, window, route, lens)


@pytest.mark.parametrize("own_positions", [False, True])
@pytest.mark.parametrize("name", list(APPENDS))
def test_append_rope_against_its_two_calls(device, name, own_positions):
    """write_kv_rope of the new token, then the decode with its query rotated in the kernel: the
    same caches bit for bit, three calls on one workspace. The output too where the rotated query
    keeps its type (fp32; more than 8 query heads a KV head); elsewhere the append keeps what
    rounding it leaves: the scores differ by u |q||k| scale at most (u = eps / 2), which moves a
    weighted mean of V by 2 |delta s| e^(2 |delta s|) max |V|, and two roundings of outputs add
    2 u of it. (The random keys' norms lie within 1.6 sqrt(D).)"""
    H, KVH, D, qt, kt, B, W, window, route = APPENDS[name]
    ws = torch.zeros(nat.lib().msattn_workspace_bytes(B, 1, H, KVH, D, W * 16), dtype=torch.uint8,
                     device=device)
    for call in range(3):
        q, k, v, kc, vc, table, lens, cos, sin, win, _, host = append_case(name, device, call)
        win = win or None
        assert kernel_route(q, kc, table, window=win) == route
        pos = (lens * 3 - 5) if own_positions else None
        a = (kc.clone(), vc.clone())
        note(f"append {name} call {call}: lens={host[:6]}")
        rope = (cos, sin) if pos is None else (cos, sin, pos)
        out = paged_attention_append(q, k, v, kc, vc, table, lens, window=win, workspace=ws,
                                     rope=rope)
        write_kv_rope(None, k, v, *a, table, lens - 1, cos, sin, pos)
        assert torch.equal(bits(kc), bits(a[0])) and torch.equal(bits(vc), bits(a[1]))
        if win is None:
            want = paged_attention(q, *a, table, lens, workspace=ws,
                                   rope=(cos, sin, lens - 1 if pos is None else pos))
        else:  # the in-kernel query rotation, then a decode under a window
            turned = write_kv_rope(q, k, v, a[0].clone(), a[1].clone(), table, lens - 1, cos, sin,
                                   pos)
            want = paged_attention(turned, *a, table, lens, window=win, workspace=ws)
        if qt == F32 or H // KVH > 8:
            assert torch.equal(out, want)
        else:
            u = torch.finfo(qt).eps / 2
            ds = u * D ** -0.5 * q.float().norm(dim=-1).max().item() * 1.6 * D ** 0.5
            bound = (2 * ds * math.exp(2 * ds) + 2 * u) * vc.float().abs().nan_to_num(0).max().item()
            assert (out.float() - want.float()).abs().max().item() <= bound
        assert out[0].abs().max() == 0  # the pad row


@pytest.mark.parametrize("name", ["C2 geometry bf16", "bf16 over fp8 D128", "fp32",
                                  "stream-K", "fp16 over fp8 D64", "head_dim 80 (two launches)",
                                  "stream-K, fp8 (two launches)", "one query head a KV head",
                                  "bf16 over fp32", "stream-K, D64"])
def test_append_rope_against_64_bits(device, name):
    """Against attention in 64 bits over the caches as they stand after the call, the query
    rotated in 64 bits. Bounds: the score error from the rotated query, kept in two parts of its
    type (relative u^2 an element, u = eps / 2; fp16's least step 2^-24, halved, a floor), is at
    most (u^2 |q| + 2^-25 sqrt(D)) |k| scale, the sums' in fp32 2^-22 |q||k| scale, and moves a
    weight by at most e^(2 |delta s|) - 1; the output's own rounding adds u; fp32's own sums 2^-20
    more. Outputs are weighted means of V, so the whole is at most
    (2 max |delta s| 1.01 + u + 2^-20) max |V|."""
    q, k, v, kc, vc, table, lens, cos, sin, _, _, host = append_case(name, device)
    note(f"64 bits {name}")
    out = paged_attention_append(q, k, v, kc, vc, table, lens, rope=(cos, sin))
    pos = torch.tensor(host)[:, None] - 1
    turned, _ = rotate64(q, cos, sin, pos)
    u = torch.finfo(q.dtype).eps / 2
    rows = [b for b in range(len(host)) if b < 6 and b != 3]  # (row 3 holds a hole)
    for b in rows:
        n = host[b]
        if n == 0:
            assert out[b].abs().max() == 0
            continue
        kk = torch.from_numpy(dense.gather_rows(kc.cpu(), table[b].cpu(), n))
        vv = torch.from_numpy(dense.gather_rows(vc.cpu(), table[b].cpu(), n))
        want = dense.attend_f64(turned[b].numpy(), kk.numpy(), vv.numpy(),
                                dense.keep_mask(n, 1, True, None), q.shape[3] ** -0.5)
        ds = ((u * u + 2.0 ** -22) * turned[b].norm(dim=-1).max() +
              (2.0 ** -25 * q.shape[3] ** 0.5 if q.dtype == F16 else 0)) * q.shape[3] ** -0.5 * \
            kk.norm(dim=-1).max()
        assert ds < 0.2
        bound = (2.02 * ds.item() * math.exp(2 * ds.item()) + u + 2.0 ** -20) * \
            vv.abs().max().item()
        err = (out[b].cpu().double() - torch.from_numpy(want)).abs().max().item()
        assert err <= bound, (b, err, bound)


def test_append_rope_unaligned_and_infinite(device):
    """New rows off 16 bytes take two launches, with the same output; an infinite query element
    makes its own row NaN or infinite and no other."""
    q, k, v, kc, vc, table, lens, cos, sin, _, _, host = append_case("stream-K", device)
    a = (kc.clone(), vc.clone())
    off = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape).copy_(t)  # noqa: E731
    note("unaligned new rows")
    out = paged_attention_append(q, k, v, kc, vc, table, lens, rope=(cos, sin))
    got = paged_attention_append(q, off(k), off(v), *a, table, lens, rope=(cos, sin))
    assert torch.equal(got, out) and torch.equal(bits(kc), bits(a[0])) and torch.equal(bits(vc), bits(a[1]))
    q2 = q.clone()
    q2[2, 0, 5, 3] = math.inf
    note("infinite query element")
    got = paged_attention_append(q2, k, v, *a, table, lens, rope=(cos, sin))
    assert not bool(got[2, 0, 5].isfinite().all())
    got[2, 0, 5] = out[2, 0, 5]
    assert torch.equal(got, out)


def test_append_partial_rotation_and_refusals(device):
    q, k, v, kc, vc, table, lens, cos, sin, _, _, host = append_case("C2 geometry bf16", device)
    c, s = tables(64 * 16, 32, device)
    a = (kc.clone(), vc.clone())
    note("partial rotation")
    out = paged_attention_append(q, k, v, kc, vc, table, lens, rope=(c, s))
    turned = write_kv_rope(q, k, v, *a, table, lens - 1, c, s)
    assert torch.equal(bits(kc), bits(a[0])) and torch.equal(out, paged_attention(turned, *a, table, lens))
    for bad in ((cos,), (cos, sin[:, :32]), (cos[:, :63], sin[:, :63]),
                (cos, sin, torch.zeros(5)), (cos.repeat(1, 2), sin.repeat(1, 2))):
        with pytest.raises(ValueError):
            paged_attention_append(q, k, v, kc, vc, table, lens, rope=bad)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("R", [64, 32])
def test_runner_rotates(device, fused, R):
    """GraphedDecodeRunner with rotation tables over several steps and batch sizes: its graph's
    outputs and caches are the eager calls'."""
    H, KVH, D, W, layers = 14, 2, 64, 8, 2
    g = torch.Generator().manual_seed(11)
    pa = PagedAttention(H, KVH, D, num_blocks=64, block_size=16, dtype=BF16, device=device,
                        kv_dtype=BF16)
    caches = [pa.allocate_kv_cache() for _ in range(layers)]
    mirror = [(a.clone(), b.clone()) for a, b in caches]
    cos, sin = tables(W * 16, R, device)
    runner = GraphedDecodeRunner([DecodeLayer(pa, *c) for c in caches], W, buckets=(1, 4, 8),
                                 fused_append=fused, rope=(cos, sin))
    perm = torch.randperm(64, generator=g)
    ctx = [0, 5, 15, 31, 100, 127, 64, 1]
    for step in range(4):
        B = (8, 3, 8, 1)[step]
        rnd = lambda n: torch.randn(layers, B, 1, n, D, generator=g).to(BF16).to(device)  # noqa: E731
        q, k, v = rnd(H), rnd(KVH), rnd(KVH)
        rows = [perm[b * W:(b + 1) * W].tolist() for b in range(B)]
        note(f"runner step {step} batch {B}")
        out = runner.decode(q, k, v, rows, ctx[:B])
        table = torch.tensor(rows, dtype=torch.int32, device=device)
        lens = torch.tensor(ctx[:B], dtype=torch.int32, device=device) + 1
        for li, (a, b) in enumerate(mirror):
            turned = write_kv_rope(q[li], k[li], v[li], a, b, table, lens - 1, cos, sin)
            want = paged_attention(turned, a, b, table, lens, max_context=W * 16)
            # (a bucket of more rows than the call may split its keys otherwise)
            assert (out[li].float() - want.float()).abs().max() <= 2.0 ** -6 * want.float().abs().max()
            assert torch.equal(a, caches[li][0]) and torch.equal(b, caches[li][1])
        ctx = [min(c + 1, W * 16 - 1) for c in ctx]
