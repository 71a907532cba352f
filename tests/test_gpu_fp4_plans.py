"""Every compiled kernel of the 4-bit cache's attention (the geometries of test_fp4_plans.py) against
64 bits: each output of each call, over contexts whose answers show every key's weight (the bound of
test_fp4_marks.py, with sum p_j |v_j - out| taken as at most sum p_j |v_j| + |out|)."""
import math

import pytest
import torch

from miniserve_amd import _native as nat, paged_attention_fp4
from test_fp4_marks import F16, F32, SCALE, Marked
from test_fp4_plans import LIST, PARTS, PLANS, lens_of, named, plan_of

pytestmark = pytest.mark.gpu
HEADER = (64 + 4096) * 4


def marked(c, holes=False):
    dtype, D, _, H, KVH, B, _, cap, q_len, bs, _, _ = c
    assert plan_of(c) == c[2]
    lens = lens_of(c)
    x = Marked(H, KVH, D, dtype, lens, q_len, bs, extra=(cap - -(-max(max(lens), 1) // bs) * bs) // bs)
    assert x.table.shape[1] * bs == cap
    if holes:
        x.table[0, lens[0] // bs // 2] = -1
    return x


def check(device, x, got, causal, window):
    f64 = torch.float64
    B, T, H, D = got.shape
    KVH = H // x.G
    q, got = x.q.to(device).to(f64), got.to(f64)
    half, least = torch.finfo(x.q.dtype).eps / 2, 2.0 ** -25 if x.q.dtype == F16 else 0.0
    a = 2.0 ** (-24 if x.q.dtype == F32 else -16)
    for b, n in enumerate(x.lens):
        if n == 0:
            assert not got[b].any()
            continue
        k, v, live = (torch.from_numpy(y).to(device) for y in x.keys(b))
        v = torch.where(live[:, None, None], v, 0.0)
        key, at = torch.arange(n, device=device), n - T + torch.arange(T, device=device)[:, None]
        keep = (key < n) & live
        keep = keep & (key <= at) if causal else keep.expand(T, n)
        if window:
            keep = keep & (key > at - window)
        step = max(1, 20_000_000 // (n * x.G))
        sums = (n / 32 + 40) * 2.0 ** -23
        for h in range(KVH):
            kh, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            for t0 in range(0, T, step):
                see = keep[t0:t0 + step, None]
                s = SCALE * (q[b, t0:t0 + step, h * x.G:(h + 1) * x.G].reshape(-1, D) @ kh)
                s = s.view(-1, x.G, n).masked_fill(~see, -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
                total = p.sum(-1, keepdim=True)
                p = (p / torch.where(total > 0, total, 1.0)).view(-1, n)
                out, mass = p @ vh, p @ vh.abs()
                most = s.masked_fill(~see, 0.0).abs().amax()
                c = torch.expm1(16 * 2.0 ** -24 * most) + 2.0 ** -18
                far = mass + out.abs()
                limit = 1.01 * (c / (1 - c) * far + a * mass + sums * far) + half * out.abs() + least
                limit = torch.where(total.view(-1, 1) > 0, limit, 0.0)
                diff = (got[b, t0:t0 + step, h * x.G:(h + 1) * x.G].reshape(-1, D) - out).abs()
                bad = ~(diff <= limit)
                assert not bad.any(), (b, h, t0, bad.nonzero()[0].tolist(), int(bad.sum()),
                                       diff[bad][0].item(), limit[bad][0].item())


@pytest.mark.parametrize("c", PLANS, ids=named)
def test_every_kernel(device, c):
    """Twice over a workspace of NaN past its header, which stays zero; bit for bit the same."""
    dtype, D, _, H, KVH, B, _, cap, q_len, _, causal, window = c
    x = marked(c, holes=PLANS.index(c) % 3 == 0)
    nbytes = nat.lib().msattn_fp4_workspace_bytes(B, q_len, H, KVH, D, cap, nat.DTYPE_CODES[dtype])
    ws = torch.full((nbytes,), 255, dtype=torch.uint8, device=device)
    args = (x.q.to(device), *(y.to(device) for y in x.caches), x.table.to(device),
            torch.tensor(x.lens, dtype=torch.int32, device=device))
    print(f"[case] plan {named(c)}", flush=True)
    outs = []
    for _ in range(2):
        ws[:HEADER], ws[HEADER:] = 0, 255
        outs.append(paged_attention_fp4(*args, causal=causal, window=window, scale=SCALE, workspace=ws))
        assert not ws[:HEADER].any()
    assert torch.equal(*outs)
    check(device, x, outs[0], causal, window)


@pytest.mark.parametrize("c", [c for c in PLANS if c[2][1] == 4 or c[2][0] in (PARTS, LIST)], ids=named)
def test_nan_of_a_value(device, c):
    """Two NaN blocks: the outputs of the queries that see their keys, in those dims; every other output
    bit for bit what it was."""
    dtype, D, _, H, KVH, B, _, _, T, bs, causal, window = c
    x = marked(c)
    n = x.lens[0]
    args = (x.table.to(device), torch.tensor(x.lens, dtype=torch.int32, device=device))
    call = lambda: paged_attention_fp4(x.q.to(device), *(y.to(device) for y in x.caches), *args,
                                       causal=causal, window=window, scale=SCALE)
    clean = call()
    want = torch.zeros(T, H, D, dtype=torch.bool)
    for key, head, block in ((n // 2, KVH - 1, 0), (n - 1, 0, D // 32 - 1)):
        page, slot = int(x.table[0, key // bs]), key % bs
        x.caches[1][page, head, slot // 16, 8 * D + 16 * block + slot % 16] = 255
        at = n - T + torch.arange(T)
        sees = (at >= key) if causal else torch.ones(T, dtype=torch.bool)
        if window:
            sees = sees & (key > at - window)
        want[sees, head * x.G:(head + 1) * x.G, 32 * block:32 * block + 32] = True
    print(f"[case] NaN {named(c)}", flush=True)
    out = call()
    want = want.to(device)
    assert torch.equal(out[0].isnan(), want) and not clean.isnan().any()
    assert torch.equal(out[1:], clean[1:]) and torch.equal(out[0][~want], clean[0][~want])
