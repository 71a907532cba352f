"""Rotated writes, shared-prefix attention and rotated appends in a row, through one workspace, each
step checked by place: the caches against the rotation in 64 bits position by position, then the
attention against 64 bits over the keys and values that the caches hold, so that only the kernel's own
error is left in the bound. Every reference is shown to notice a lost newest key, two values in each
other's places, a skipped page and an output of zeros before the kernel is compared.

Bounds. A written key is off by 2^-22 (|a c| + |b s|) from the rotation in fp32 and by half a step of
its type (see test_gpu_rope_write); values and positions not written are equal bit for bit. For the
attention, with p the weights in 64 bits and out = sum p_j v_j, the kernel's weights are off by
factors within 1 +- E, E = u + (e^(2 ds) - 1) + 2^-18: u = eps / 2 rounds them to the query type, 2^-18
is the hardware's 2^x and its argument's rounding, ds bounds a score's error: (D + 8) 2^-24 |q||k|
scale, and where the append rotates the query, kept in two parts of its type, (u^2 + 2^-22) |q||k|
scale more (fp16: 2^-25 sqrt(D) |k| scale for its least step). Divided by a sum of the rounded weights or
of the unrounded ones: at most E / (1 - E) (sum p_j |v_j| + |out|). fp16 weights below 2^-14 are off by
2^-25 beside a largest one of 1 or more: 2^-25 sum |v_j - out| / L. The sums in fp32 add (n / 16 + 64)
2^-24 of sum p_j |v_j| + |out|, the output's rounding u |out| and half of fp16's least step.
"""
import math

import pytest
import torch

from miniserve_amd import (_native as nat, paged_attention_append, paged_attention_shared,
                           write_kv_rope)
from test_gpu_rope_write import SUBNORMAL

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def note(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


def rotate64(x, cos, sin, first):
    """(rotated, |a c| + |b s|) of x [tokens, heads, D] at positions first .. in 64 bits."""
    x, half = x.double(), x.shape[-1] // 2
    c, s = (t[first:first + len(x)].double()[:, None] for t in (cos, sin))
    turned = torch.cat((-x[..., half:], x[..., :half]), -1)
    return x * c + turned * s, (x * c).abs() + (turned * s).abs()


def rounded_bound(y, size, dtype):
    half = torch.finfo(dtype).eps / 2
    return half * y.abs() * (1 + half) + SUBNORMAL[dtype] / 2 + 2.0 ** -22 * size


def attend(q, k, v, dtype, split, bs):
    """(output, bound) [T, H, D] of the last T queries of a sequence in 64 bits; what a mistake would
    change is checked to exceed twice the bound."""
    T, H, D = q.shape
    n, KVH = k.shape[:2]
    u, scale = torch.finfo(dtype).eps / 2, D ** -0.5
    out, bound = torch.zeros(T, H, D).double(), torch.zeros(T, H, D).double()
    mutants = {}
    for kvh in range(KVH):
        heads = slice(kvh * (H // KVH), (kvh + 1) * (H // KVH))
        rows, kk, vv = q[:, heads].reshape(-1, D), k[:, kvh], v[:, kvh]
        last = torch.arange(n - T, n).repeat_interleave(H // KVH)
        seen = torch.arange(n) <= last[:, None]
        x = (rows @ kk.T * scale).masked_fill(~seen, -math.inf)
        w = torch.exp(x - x.amax(1, keepdim=True))
        L = w.sum(1, keepdim=True)
        p = w / L
        o = p @ vv
        size = p @ vv.abs() + o.abs()
        norm = kk.norm(dim=1).max() * scale
        ds = (D + 8) * 2.0 ** -24 * rows.norm(dim=1) * norm
        if split:
            ds = ds + (u * u + 2.0 ** -22) * rows.norm(dim=1) * norm
            ds = ds + (2.0 ** -25 * D ** 0.5 * norm if dtype == F16 else 0)
        E = (u + torch.expm1(2 * ds) + 2.0 ** -18)[:, None]
        e = E / (1 - E) * size + (n / 16 + 64) * 2.0 ** -24 * size + u * o.abs() * (1 + u)
        if dtype == F16:
            far = torch.stack([seen[r].double() @ (vv - o[r]).abs() for r in range(len(p))])
            e = e + 2.0 ** -25 * far / L + 2.0 ** -25
        out[:, heads], bound[:, heads] = o.view(T, -1, D), e.view(T, -1, D)

        def without(gone):  # the output over the other keys
            left = w * ~gone
            return left @ vv / left.sum(1, keepdim=True).clamp(min=1e-300)

        every = torch.arange(n)
        swapped = vv.clone()
        swapped[[n - T - 1, n // 2]] = vv[[n // 2, n - T - 1]]
        for what, y in (("newest key", without(every == last[:, None])),
                        ("swapped values", p @ swapped),
                        ("first page", without((every < bs).expand(len(p), n))),
                        ("last full page", without(((every >= (n // bs - 1) * bs) & (every < n // bs * bs)).expand(len(p), n))),
                        ("zeros", torch.zeros_like(o))):
            shows = bool(((y - o).abs() > 2 * e).any())
            mutants[what] = mutants.get(what, False) or shows
    assert all(mutants.values()), f"a mistake would not show: {mutants}"
    return out, bound


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("H,KVH,D,dtype", [(14, 2, 64, BF16), (8, 2, 128, F16)])
def test_every_step_by_place(device, H, KVH, D, dtype, graph):
    g = torch.Generator().manual_seed(3 * H + D)
    bs, W = 16, 20
    members, prefix = [3, 2], [7, 4]  # rows and pages of the two groups; a loose row last
    B = sum(members) + 1
    rows = [0, members[0], sum(members)]
    inv = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
    a = torch.arange(W * bs, dtype=torch.float64)[:, None] * inv
    cos, sin = (torch.cat((f(a), f(a)), -1).float() for f in (torch.cos, torch.sin))
    dcos, dsin = cos.to(device), sin.to(device)
    perm = torch.randperm(B * W, generator=g).tolist()
    kc, vc = (torch.full((B * W, bs, KVH, D), math.nan, dtype=dtype, device=device) for _ in range(2))
    ws = torch.zeros(nat.lib().msattn_shared_workspace_bytes(B, 8, H, KVH, D, W * bs, 2),
                     dtype=torch.uint8, device=device)
    draw = lambda *n: torch.randn(*n, D, generator=g).to(dtype)  # noqa: E731
    table = torch.full((B, W), -1, dtype=torch.int32)
    held = [[torch.empty(0, KVH, D, dtype=dtype)] * 2 for _ in range(B)]  # the caches by position

    def written(b, k, v, start):
        """Row b's tokens k, v at start ..: read back, checked; what stood before, unchanged."""
        n = start + len(k)
        pages = table[b, :-(-n // bs)].long().to(device)
        got = [c[pages].cpu().reshape(-1, KVH, D)[:n] for c in (kc, vc)]
        for old, new in zip(held[b], got):
            assert torch.equal(old[:start], new[:start])
        y, size = rotate64(k, cos, sin, start)
        assert bool(((got[0][start:].double() - y).abs() <= rounded_bound(y, size, dtype)).all())
        assert torch.equal(got[1][start:], v)
        held[b] = got

    for i, (n, pages) in enumerate(zip(members, prefix)):
        ids = [perm.pop() for _ in range(pages)]
        table[rows[i]:rows[i] + n, :pages] = torch.tensor(ids, dtype=torch.int32)
        k, v = draw(1, pages * bs, KVH), draw(1, pages * bs, KVH)
        note(f"prefix {i}")
        write_kv_rope(None, k.to(device), v.to(device), kc, vc, torch.tensor([ids], dtype=torch.int32),
                      0, dcos, dsin)
        for b in range(rows[i], rows[i] + n):
            written(b, k[0], v[0], 0)
    for b in range(B):
        for c in range(W):
            if table[b, c] < 0:
                table[b, c] = perm.pop()
    dtable = table.to(device)
    drows, dpages = (torch.tensor(x, dtype=torch.int32, device=device) for x in (rows, prefix))
    s = {}

    def several(T):  # T tokens a row written, then attended: the two calls
        q = write_kv_rope(s["q"], s["k"], s["v"], kc, vc, dtable, s["start"], dcos, dsin)
        return q, paged_attention_shared(q, kc, vc, dtable, s["start"] + T, drows, dpages,
                                         max_context=W * bs, workspace=ws)

    def one(T):  # one token a row: the append
        return None, paged_attention_append(s["q"], s["k"], s["v"], kc, vc, dtable, s["start"] + 1,
                                            max_context=W * bs, workspace=ws, rope=(dcos, dsin))

    graphs = {}

    def step(fn, T, start):
        q, k, v = draw(B, T, H), draw(B, T, KVH), draw(B, T, KVH)
        key = (fn, T)
        if not graph or key not in graphs:
            s.update(q=q.to(device), k=k.to(device), v=v.to(device),
                     start=torch.tensor(start, dtype=torch.int32, device=device))
            turned, out = fn(T)
            if graph:  # captured on buffers of its own, replayed from the second such step on
                kept, captured = dict(s), torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    outs = fn(T)
                graphs[key] = (kept, captured, outs)
        else:
            kept, captured, (turned, out) = graphs[key]
            for name, x in (("q", q), ("k", k), ("v", v), ("start", torch.tensor(start))):
                kept[name].copy_(x)
            captured.replay()
        for b in range(B):
            written(b, k[b], v[b], start[b])
            y, size = rotate64(q[b], cos, sin, start[b])
            if turned is not None:  # the query that the attention was given
                given = turned[b].cpu().double()
                assert bool(((given - y).abs() <= rounded_bound(y, size, dtype)).all())
                y = given
            want, bound = attend(y, *(x.double() for x in held[b]), dtype, turned is None, bs)
            over = ((out[b].cpu().double() - want).abs() - bound).max().item()
            assert over <= 0, f"row {b} at {start[b]}: {over:.3e} over the bound"

    start = [len(x[0]) for x in held]
    start[-1] = 40  # the loose row's prompt
    k, v = draw(1, 40, KVH), draw(1, 40, KVH)
    write_kv_rope(None, k.to(device), v.to(device), kc, vc, dtable[-1:], 0, dcos, dsin)
    written(B - 1, k[0], v[0], 0)
    for turn in range(3):
        note(f"chunk {turn}")
        step(several, 8, start)
        start = [n + 8 for n in start]
        for _ in range(2):
            note(f"decode {turn}")
            step(one, 1, start)
            start = [n + 1 for n in start]
        note(f"draft {turn}")
        step(several, 4, start)
        start = [n + 1 + (b + turn) % 4 for b, n in enumerate(start)]  # so many of the drafts stay
        note(f"decode behind every prefix {turn}")
        step(several, 1, start)
        start = [n + 1 for n in start]
