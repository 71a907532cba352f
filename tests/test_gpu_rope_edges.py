"""Rotated writes and appends at the ends of what their arguments allow."""
import math

import pytest
import torch

import test_gpu_rope_write as base
from miniserve_amd import (PagedAttention, attention, kernel_route, paged_attention_append,
                           write_kv_rope)
from miniserve_amd.graphs import DecodeLayer, GraphedDecodeRunner
from oracle import dense
from test_gpu_serving_places import attend

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
note, tables, rotate64, bits = base.note, base.tables, base.rotate64, base.bits


@pytest.mark.parametrize("form", ["rows", "tokens", "int"])
def test_positions_past_32_bits_are_clamped(device, form):
    """int64 positions past int32 are the tables' last row, or their first, as any position outside
    is; they are not taken modulo 2^32."""
    g = torch.Generator().manual_seed(5)
    B, T, H, KVH, D, bs, W = 3, 18, 4, 2, 64, 16, 2
    q, k, v = base.sources(H, KVH, D, F16, B, T, "fused", g, device)
    kc, vc = base.pool(B * W, bs, KVH, D, F16, g, device)
    kc0, vc0 = kc.clone(), vc.clone()
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32)
    cos, sin = tables(50, D, device)
    wide = torch.tensor([2 ** 31, 2 ** 40 + 7, -2 ** 33 + 5])
    last = torch.tensor([49, 49, 0])
    given, full = {
        "rows": (wide, None),
        "tokens": (wide[:, None].expand(B, T), last[:, None].expand(B, T)),
        "int": (2 ** 32 + 3, torch.full((B, T), 49)),
    }[form]
    if full is None:  # (the first tokens' positions; the others follow)
        full = (wide[:, None].clamp(-2 ** 31, 2 ** 31 - 1) + torch.arange(T))
    note(f"positions past 32 bits, {form}")
    out = write_kv_rope(q, k, v, kc, vc, table.to(device), [2, 0, 5], cos, sin,
                        given.to(device) if isinstance(given, torch.Tensor) else given)
    base.check_write(q, k, v, kc0, vc0, kc, vc, out, table, [2, 0, 5], cos, sin, full)


def test_starts_past_32_bits_write_nothing(device):
    """int64 starts past int32 lie outside every table: their tokens are rotated, not written."""
    g = torch.Generator().manual_seed(6)
    B, T, H, KVH, D, bs, W = 4, 5, 2, 2, 64, 16, 2
    q, k, v = base.sources(H, KVH, D, BF16, B, T, "dense", g, device)
    kc, vc = base.pool(B * W, bs, KVH, D, BF16, g, device)
    kc0, vc0 = kc.clone(), vc.clone()
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32)
    cos, sin = tables(40, D, device)
    start = [2 ** 32 + 3, 4, -2 ** 32 + 2, 2 ** 31]
    note("starts past 32 bits")
    out = write_kv_rope(q, k, v, kc, vc, table.to(device), torch.tensor(start, device=device), cos, sin)
    base.check_write(q, k, v, kc0, vc0, kc, vc, out, table, start, cos, sin)


def test_append_positions_past_32_bits(device):
    q, k, v, kc, vc, table, lens, cos, sin, _, _, host = base.append_case("C2 geometry bf16", device)
    a = (kc.clone(), vc.clone())
    wide = torch.tensor([2 ** 32 + 5, 2 ** 31, -2 ** 32 + 9, 7] * 8, device=device)
    near = wide.clamp(0, cos.shape[0] - 1).to(torch.int32)
    note("append, positions past 32 bits")
    out = paged_attention_append(q, k, v, kc, vc, table, lens, rope=(cos, sin, wide))
    want = paged_attention_append(q, k, v, *a, table, lens, rope=(cos, sin, near))
    assert torch.equal(out, want) and torch.equal(bits(kc), bits(a[0]))


@pytest.mark.parametrize("name", ["C2 geometry bf16", "stream-K", "bf16 over fp32",
                                  "two query heads a KV head", "stream-K, D64"])
def test_append_over_an_infinite_key(device, name):
    """A cached key whose one element is -inf, and queries that are positive there: its score is
    -inf and it weighs nothing, as in the two calls; queries that are negative there have no finite
    answer. The bound is that of the appends against 64 bits: the query in two parts of its type
    (u^2, fp16's least step), the sums in fp32, the output's rounding."""
    q, k, v, kc, vc, table, lens, cos, sin, _, _, host = base.append_case(name, device)
    H, KVH, D = q.shape[2], kc.shape[2], q.shape[3]
    pos, row, dim = torch.tensor(host)[:, None] - 1, 2, 3  # (row 2 fills its table)
    sign = rotate64(q, cos, sin, pos)[0][row, 0, :, dim].sign()
    flip = torch.ones(H).double()
    flip[H - 1] = -1.0  # the last head's score is +inf
    q[row, 0] *= (sign * flip).to(q.dtype).to(device)[:, None]
    turned, _ = rotate64(q, cos, sin, pos)
    bad = 37
    page = int(table[row, bad // 16])
    kc[page, bad % 16, :, dim] = -math.inf
    note(f"infinite key, {name}")
    out = paged_attention_append(q, k, v, kc, vc, table, lens, rope=(cos, sin))[row].cpu().double()
    n = host[row]
    kk = torch.from_numpy(dense.gather_rows(kc.cpu(), table[row].cpu(), n, q.dtype))
    vv = torch.from_numpy(dense.gather_rows(vc.cpu(), table[row].cpu(), n, q.dtype))
    kk[bad] = 0
    keep = dense.keep_mask(n, 1, True, None)
    keep[:, bad] = False
    want = torch.from_numpy(dense.attend_f64(turned[row].numpy(), kk.numpy(), vv.numpy(), keep, D ** -0.5))
    u = torch.finfo(q.dtype).eps / 2
    ds = (((u * u + 2.0 ** -22) * turned[row].norm(dim=-1).max() +
           (2.0 ** -25 * D ** 0.5 if q.dtype == F16 else 0)) * D ** -0.5 * kk.norm(dim=-1).max()).item()
    bound = (2.02 * ds * math.exp(2 * ds) + 4 * u + 2.0 ** -18 +
             (n * 2.0 ** -24 if q.dtype == F16 else 0)) * vv.abs().max().item()
    assert (out - want)[:, :H - 1].abs().max().item() <= bound
    assert not bool(out[:, H - 1].isfinite().any())


@pytest.mark.parametrize("name", ["C2 geometry bf16", "fp32", "stream-K, fp8 (two launches)",
                                  "head_dim 80 (two launches)"])
def test_append_takes_tables_off_16_bytes(device, name):
    q, k, v, kc, vc, table, lens, cos, sin, _, _, _ = base.append_case(name, device)
    a = (kc.clone(), vc.clone())
    off = lambda t: torch.empty(t.numel() + 1, device=device)[1:].view(t.shape).copy_(t)  # noqa: E731
    note(f"tables off 16 bytes, {name}")
    want = paged_attention_append(q, k, v, *a, table, lens, rope=(cos, sin))
    out = paged_attention_append(q, k, v, kc, vc, table, lens, rope=(off(cos), off(sin)))
    assert torch.equal(out, want) and torch.equal(bits(kc), bits(a[0]))


def runner_of(device, W, rope, H=14, KVH=2, D=64, fused=True):
    pa = PagedAttention(H, KVH, D, num_blocks=16, block_size=16, dtype=BF16, device=device,
                        kv_dtype=BF16)
    caches = pa.allocate_kv_cache()
    return GraphedDecodeRunner([DecodeLayer(pa, *caches)], W, buckets=(1, 2), fused_append=fused,
                               rope=rope), caches


@pytest.mark.parametrize("fused", [True, False])
def test_runner_refuses_positions_past_its_tables(device, fused):
    """A context longer than the rotation tables has no position there: the step is refused before
    it writes; one that fits runs."""
    cos, sin = tables(40, 64, device)
    runner, caches = runner_of(device, 4, (cos, sin), fused=fused)
    g = torch.Generator().manual_seed(3)
    rnd = lambda n: torch.randn(1, 2, 1, n, 64, generator=g).to(BF16).to(device)  # noqa: E731
    q, k, v = rnd(14), rnd(2), rnd(2)
    rows = [[0, 1, 2, 3], [4, 5, 6, 7]]
    note("positions past the tables")
    for ctx in ([3, 40], [63, 0]):
        with pytest.raises(ValueError, match="rotation tables"):
            runner.decode(q, k, v, rows, ctx)
        assert not bits(caches[0]).any() and not bits(caches[1]).any()
    out = runner.decode(q, k, v, rows, [3, 39])
    a = [torch.zeros_like(c) for c in caches]
    lens = torch.tensor([4, 40], dtype=torch.int32, device=device)
    write_kv_rope(q[0], k[0], v[0], *a, torch.tensor(rows, dtype=torch.int32, device=device),
                  lens - 1, cos, sin)
    assert torch.equal(caches[0], a[0]) and torch.equal(caches[1], a[1]) and bool(out.isfinite().all())


def test_runner_takes_tables_off_16_bytes(device):
    cos, sin = tables(64, 64, device)
    off = lambda t: torch.empty(t.numel() + 1, device=device)[1:].view(t.shape).copy_(t)  # noqa: E731
    g = torch.Generator().manual_seed(4)
    rnd = lambda n: torch.randn(1, 2, 1, n, 64, generator=g).to(BF16).to(device)  # noqa: E731
    q, k, v = rnd(14), rnd(2), rnd(2)
    rows = [[0, 1, 2, 3], [4, 5, 6, 7]]
    note("runner, tables off 16 bytes")
    got = [runner_of(device, 4, r)[0].decode(q, k, v, rows, [3, 39]) for r in ((cos, sin), (off(cos), off(sin)))]
    assert torch.equal(*got)


def test_partial_rotation_on_another_device_than_the_current_one(device, monkeypatch):
    """Every launch of an append with a rotary size below head_dim runs with the tensors' device
    current: here the current one is reported as another, and entering a device is recorded."""
    q, k, v, kc, vc, table, lens, _, _, _, _, _ = base.append_case("C2 geometry bf16", device)
    cos, sin = tables(64 * 16, 32, device)
    inside = []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            inside.append(self.dev)

        def __exit__(self, *e):
            inside.pop()

    seen = []
    real_write, real_attend = attention.write_kv_rope, attention.paged_attention
    monkeypatch.setattr(attention, "write_kv_rope", lambda *a, **kw: (seen.append(list(inside)), real_write(*a, **kw))[1])
    monkeypatch.setattr(attention, "paged_attention", lambda *a, **kw: (seen.append(list(inside)), real_attend(*a, **kw))[1])
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", Device)
    note("another device")
    paged_attention_append(q, k, v, kc, vc, table, lens, rope=(cos, sin))
    assert seen[-1] == [device] and len(seen) == 2 and not inside


def test_more_tokens_than_a_launch_holds_waves(device):
    """2^26 + 8 tokens: a wave each would be a launch of more than 2^32 threads."""
    T, D = 2 ** 26 + 8, 16
    g = torch.Generator().manual_seed(12)
    some = torch.randn(2 ** 16, 1, D, generator=g).to(BF16).to(device)
    q = some.repeat(2 ** 10 + 1, 1, 1)[None, :T]
    k = some[:1].expand(1, T, 1, D)
    kc, vc = base.pool(2, 16, 1, D, BF16, g, device)
    kc0, vc0 = kc.clone(), vc.clone()
    cos, sin = tables(3, D, device)
    note("more than 2^26 tokens")
    out = write_kv_rope(q, k, k, kc, vc, torch.tensor([[-1]], dtype=torch.int32, device=device), 0,
                        cos, sin)
    x = some.float()
    turned = torch.cat((-x[..., D // 2:], x[..., :D // 2]), -1)
    for t in range(2):  # (positions 0 and 1; all others are past the tables: their last row)
        y = (x[t] * cos[t] + turned[t] * sin[t]).to(BF16)
        assert torch.equal(out[0, t], y)
    y = (x * cos[2] + turned * sin[2]).to(BF16)
    for t in range(0, T, 2 ** 16):
        n = min(2 ** 16, T - t)
        lo = 2 if t == 0 else 0
        assert torch.equal(out[0, t + lo:t + n], y[lo:n])
    assert torch.equal(kc, kc0) and torch.equal(vc, vc0)


@pytest.mark.parametrize("rope", [False, True])
def test_append_refuses_what_lies_elsewhere(device, rope):
    """New rows, caches, output and workspace that the kernels could not address."""
    q, k, v, kc, vc, table, lens, cos, sin, _, _, _ = base.append_case("C2 geometry bf16", device)
    a = (kc.clone(), vc.clone())
    B, _, H, D = q.shape
    ok = dict(k=k, v=v, kc=kc, vc=vc, out=None, workspace=None)
    bytes_ = 64 << 20
    note("operands elsewhere")
    for bad in (dict(k=k.cpu()), dict(v=v.cpu()), dict(out=torch.empty(B, 1, H, D, dtype=BF16)),
                dict(out=torch.empty(B - 1, 1, H, D, dtype=BF16, device=device)),
                dict(out=torch.empty(B, 1, H, D, device=device)),
                dict(out=torch.empty(B, 1, D, H, dtype=BF16, device=device).transpose(2, 3)),
                dict(workspace=torch.zeros(bytes_, dtype=torch.uint8)),
                dict(workspace=torch.zeros(2 * bytes_, dtype=torch.uint8, device=device)[::2])):
        x = dict(ok, **bad)
        with pytest.raises(ValueError, match="device|out must"):
            paged_attention_append(q, x["k"], x["v"], x["kc"], x["vc"], table, lens, out=x["out"],
                                   workspace=x["workspace"], rope=(cos, sin) if rope else None)
    assert torch.equal(bits(kc), bits(a[0])) and torch.equal(bits(vc), bits(a[1]))


@pytest.mark.parametrize("qt", [BF16, F16])
def test_generic_append_of_many_query_heads(device, qt):
    """16 query heads a KV head at head_dim 80, the generic kernel: it keeps the rotated query in fp32
    whatever the heads, so that the bound of the query in two parts holds."""
    g = torch.Generator().manual_seed(13)
    B, H, KVH, D, bs, W = 4, 32, 2, 80, 16, 16
    kc, vc = base.pool(B * W, bs, KVH, D, qt, g, device)
    table = torch.randperm(B * W, generator=g).view(B, W).to(torch.int32)
    host = [37, 256, 100, 18]
    lens = torch.tensor(host, dtype=torch.int32, device=device)
    q, k, v = (torch.randn(B, 1, n, D, generator=g).to(qt).to(device) for n in (H, KVH, KVH))
    cos, sin = tables(W * bs, D, device)
    assert kernel_route(q, kc, table) == "generic"
    note(f"generic, 16 heads a KV head, {qt}")
    out = paged_attention_append(q, k, v, kc, vc, table.to(device), lens, rope=(cos, sin)).cpu().double()
    turned, _ = rotate64(q, cos, sin, torch.tensor(host)[:, None] - 1)
    for b, n in enumerate(host):
        kk, vv = (torch.from_numpy(dense.gather_rows(c.cpu(), table[b], n)) for c in (kc, vc))
        want, bound = attend(turned[b], kk, vv, qt, True, bs)
        assert ((out[b] - want).abs() - bound).max().item() <= 0
