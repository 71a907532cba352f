"""A run of the rotated writes, the shared-prefix attention and the rotated decode appends together,
as a server makes it: two system prompts written once, sequences behind them prefilled in a chunk,
decoded, drafted ahead and taken back, through one workspace. Against attention in 64 bits over the
tokens themselves, so that a key or value in a wrong place shows.

Tolerance. Of a weighted mean of V with weights from scores s: a score error of at most d moves it
by 2 d e^(2 d) max |V|. The keys are rotated in fp32 (2^-22 (|a c| + |b s|), at most 2^-21.5 |k|)
and rounded to the cache's type (u = eps / 2 relative), the query to its type in the two-call steps
(u), and sums of D products are exact to (D + 8) 2^-24, so that d <= (2 u + u^2 + 2^-20 + (D + 8)
2^-24) |q||k| scale. The values and the outputs are rounded (u each), the weights to the query type
(u, or half of fp16's least step a key), and a mean of rounded weights' own sums add 2^-18.
"""
import math

import pytest
import torch

from miniserve_amd import (_native as nat, paged_attention_append, paged_attention_shared,
                           write_kv_rope)
from oracle import dense

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def note(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


def rotate64(x, inv, first):
    """x [tokens, heads, D] rotated at positions first, first + 1, .. in 64 bits."""
    x, half = x.double(), x.shape[-1] // 2
    a = (first + torch.arange(x.shape[0], dtype=torch.float64))[:, None] * inv
    c, s = (f(torch.cat((a, a), -1)).float().double()[:, None] for f in (torch.cos, torch.sin))
    return x * c + torch.cat((-x[..., half:], x[..., :half]), -1) * s


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("H,KVH,D,dtype", [(14, 2, 64, BF16), (8, 2, 128, F16)])
def test_prefill_decode_draft(device, H, KVH, D, dtype, graph):
    g = torch.Generator().manual_seed(H + D)
    bs, W = 16, 20
    members, prefix = [3, 2], [7, 4]           # rows and pages of the two groups; a loose row last
    B = sum(members) + 1
    rows = [0, members[0], sum(members)]
    inv = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) * 2 / D)
    a = torch.arange(W * bs, dtype=torch.float64)[:, None] * inv
    cos, sin = (torch.cat((f(a), f(a)), -1).float().to(device) for f in (torch.cos, torch.sin))
    perm = torch.randperm(B * W, generator=g).tolist()
    kc, vc = (torch.full((B * W, bs, KVH, D), math.nan, dtype=dtype, device=device) for _ in range(2))
    ws = torch.zeros(nat.lib().msattn_shared_workspace_bytes(B, 8, H, KVH, D, W * bs, 2),
                     dtype=torch.uint8, device=device)
    table = torch.full((B, W), -1, dtype=torch.int32)
    K, V = [None] * B, [None] * B              # each sequence's keys (rotated, 64 bits) and values
    draw = lambda *n: torch.randn(*n, D, generator=g).to(dtype)  # noqa: E731
    for i, (n, pages) in enumerate(zip(members, prefix)):
        ids = [perm.pop() for _ in range(pages)]
        k, v = draw(1, pages * bs, KVH), draw(1, pages * bs, KVH)
        table[rows[i]:rows[i] + n, :pages] = torch.tensor(ids, dtype=torch.int32)
        note(f"prefix {i}")
        write_kv_rope(None, k.to(device), v.to(device), kc, vc, torch.tensor([ids], dtype=torch.int32),
                      0, cos, sin)
        for b in range(rows[i], rows[i] + n):
            K[b], V[b] = rotate64(k[0], inv, 0), v[0].double()
    K[-1], V[-1] = torch.empty(0, KVH, D).double(), torch.empty(0, KVH, D).double()
    for b in range(B):
        for c in range(W):
            if table[b, c] < 0:
                table[b, c] = perm.pop()
    dev_table = table.to(device)
    dev_rows, dev_pages = (torch.tensor(x, dtype=torch.int32, device=device) for x in (rows, prefix))

    def append(k, v, start):
        for b in range(B):
            K[b] = torch.cat((K[b][:start[b]], rotate64(k[b], inv, start[b])))
            V[b] = torch.cat((V[b][:start[b]], v[b].double()))

    def check(out, q, start):
        u, T = torch.finfo(dtype).eps / 2, q.shape[1]
        for b in range(B):
            n = start[b] + T
            turned = rotate64(q[b], inv, start[b])
            want = dense.attend_f64(turned.numpy(), K[b].numpy(), V[b].numpy(),
                                    dense.keep_mask(n, T, True, None), D ** -0.5)
            d = (2 * u + u * u + 2.0 ** -20 + (D + 8) * 2.0 ** -24) * D ** -0.5 * \
                (turned.norm(dim=-1).max() * K[b].norm(dim=-1).max()).item()
            bound = (2 * d * math.exp(2 * d) + 4 * u + 2.0 ** -18 +
                     (n * 2.0 ** -24 if dtype == F16 else 0)) * V[b].abs().max().item()
            err = (out[b].cpu().double() - torch.from_numpy(want)).abs().max().item()
            assert err <= bound, (b, n, err, bound)

    state = {}

    def several(T):  # T tokens a row written, then attended: the two calls
        s = state
        q = write_kv_rope(s["q"], s["k"], s["v"], kc, vc, dev_table, s["start"], cos, sin)
        return paged_attention_shared(q, kc, vc, dev_table, s["start"] + T, dev_rows, dev_pages,
                                      max_context=W * bs, workspace=ws)

    def one(T):  # one token a row: the append
        s = state
        return paged_attention_append(s["q"], s["k"], s["v"], kc, vc, dev_table, s["start"] + 1,
                                      max_context=W * bs, workspace=ws, rope=(cos, sin))

    graphs = {}

    def step(fn, T, start):
        q, k, v = draw(B, T, H), draw(B, T, KVH), draw(B, T, KVH)
        append(k, v, start)
        key = (fn, T)
        if not graph or key not in graphs:
            state.update(q=q.to(device), k=k.to(device), v=v.to(device),
                         start=torch.tensor(start, dtype=torch.int32, device=device))
            out = fn(T)
            if graph:  # captured on buffers of its own, replayed from the second such step on
                kept, captured = dict(state), torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    graph_out = fn(T)
                graphs[key] = (kept, captured, graph_out)
        else:
            kept, captured, out = graphs[key]
            for name, x in (("q", q), ("k", k), ("v", v), ("start", torch.tensor(start))):
                kept[name].copy_(x)
            captured.replay()
        check(out, q, start)

    start = [x.shape[0] for x in K]
    for turn in range(3):
        note(f"chunk {turn}")
        step(several, 8, start)
        start = [s + 8 for s in start]
        for _ in range(2):
            note(f"decode {turn}")
            step(one, 1, start)
            start = [s + 1 for s in start]
        note(f"draft {turn}")
        step(several, 4, start)
        start = [s + 1 + (b + turn) % 4 for b, s in enumerate(start)]  # so many of the drafts stay
        note(f"decode behind every prefix {turn}")
        step(several, 1, start)
        start = [s + 1 for s in start]
