"""The 4-bit paged cache on the GPU: written and read back bit for bit, attended over against 64 bits.

Tolerance of the attention. The cache's values are exact. Scores are fp32 sums of exact products:
off by at most |ds| = (P D + 8) 2^-24 scale |q||k| (P products of bf16 parts a dim, their additions,
the scale), so a weight is off by a factor e^(2 |ds|). The weights of a bf16 query are rounded once,
in numerator and sum alike (u = 2^-8); of an fp16 one they lose at most 2^-15 to its two parts, of an
fp32 one nothing. Sums over n keys go in steps of 32: (n / 32 + 40) 2^-23; the hardware's 2^x, its
argument and the joins 2^-18, as for the 16-bit caches. The output is rounded once. Outputs are
weighted means of V: the whole is at most
(4.04 |ds| e^(2 |ds|) + 3 u [bf16; else 2 u + 2^-15] + (n / 32 + 40) 2^-23 + 2^-18) max |V|.
"""
import math

import numpy as np
import pytest
import torch

from miniserve_amd import (PagedAttention, _native as nat, allocate_fp4_cache, paged_attention_fp4,
                           read_kv_fp4, write_kv_fp4)
from miniserve_amd.graphs import DecodeLayer, GraphedDecodeRunner
from oracle import dense, fp4

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def note(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


def tables(lens, bs, extra=0, seed=0, spare=3):
    """(int32 table, pages): every row's pages apart, shuffled, -1 past its end."""
    g = torch.Generator().manual_seed(seed)
    W = max(1, max(-(-n // bs) for n in lens)) + extra
    need = sum(-(-max(n, 0) // bs) for n in lens) + spare
    perm = torch.randperm(need, generator=g).tolist()
    t = torch.full((len(lens), W), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for c in range(-(-max(n, 0) // bs)):
            t[b, c] = perm.pop()
    return t, need


def storing(x, cache, table, start, is_values):
    """`cache` (uint8, CPU) with x [batch, tokens, heads, D] stored at start[b] + t, by the oracle."""
    codes, scale = fp4.unpack(cache, is_values)
    new_codes, new_scale = fp4.quantise(x)
    nb, bs = codes.shape[:2]
    for b in range(x.shape[0]):
        for t in range(x.shape[1]):
            pos = int(start[b]) + t
            if pos < 0 or pos >= table.shape[1] * bs:
                continue
            page = int(table[b, pos // bs])
            if 0 <= page < nb:
                codes[page, pos % bs], scale[page, pos % bs] = new_codes[b, t], new_scale[b, t]
    return fp4.pack(codes, scale, is_values)


# type, KV heads, D, block size, tokens, starts
STORES = [
    (BF16, 2, 64, 16, 1, [0, 15, 16, 100, -1]), (BF16, 8, 128, 16, 37, [3, 0, 250]),
    (F16, 4, 128, 32, 16, [16, 5]), (F32, 3, 96, 64, 70, [60, -5]), (F32, 1, 256, 16, 3, [31, 14]),
    (BF16, 5, 32, 48, 49, [47]), (F16, 7, 160, 16, 2, [0, 1, 2, 3, 4, 5, 6]),
    (BF16, 40, 256, 16, 2, [15, 7]), (F16, 1, 224, 16, 130, [1]),
]


@pytest.mark.parametrize("case", STORES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("views", [False, True])
def test_store_is_bit_exact(device, case, views):
    dtype, KVH, D, bs, T, starts = case
    g = torch.Generator().manual_seed(D + T)
    lens = [max(0, s + T) for s in starts]
    table, need = tables(lens, bs, extra=1, seed=T)
    if len(starts) > 1:
        table[1, 0], table[0, table.shape[1] - 1] = need + 5, 2 ** 31 - 1  # not pages
    size = (len(starts), T, KVH, D)
    if views:  # slices of a projection, heads before tokens
        both = torch.randn(size[0], 2, KVH, T, D, generator=g).to(dtype)
        k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    else:
        k, v = (torch.randn(size, generator=g).to(dtype) for _ in range(2))
    fill = [torch.randint(0, 256, (need, KVH, bs // 16, 17 * D // 2), generator=g, dtype=torch.uint8)
            for _ in range(2)]
    kc, vc = (x.to(device) for x in fill)
    kd, vd = (both.to(device)[:, i].transpose(1, 2) for i in range(2)) if views else \
        (k.to(device), v.to(device))
    note(f"store {case} views={views}")
    write_kv_fp4(kd, vd, kc, vc, table.to(device), starts)
    assert torch.equal(kc.cpu(), storing(k, fill[0], table, starts, False))
    assert torch.equal(vc.cpu(), storing(v, fill[1], table, starts, True))
    for out_type in (BF16, F32, F16):
        rk, rv = read_kv_fp4(kc, vc, table.to(device), torch.tensor(starts, device=device), T,
                             dtype=out_type)
        for cache, got, is_values in ((kc, rk, False), (vc, rv, True)):
            all_values = torch.from_numpy(fp4.values(*fp4.unpack(cache, is_values)))
            for b in range(len(starts)):
                for t in range(T):
                    pos = starts[b] + t
                    page = int(table[b, pos // bs]) if 0 <= pos < table.shape[1] * bs else -1
                    want = all_values[page, pos % bs].to(out_type) if 0 <= page < need else \
                        torch.zeros(KVH, D, dtype=out_type)
                    assert torch.equal(got[b, t].cpu(), want), (out_type, b, t)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_special_values(device, dtype):
    """Ties, the borders of the powers, subnormals, the largest numbers, infinities and NaN."""
    rows = []
    tie = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]
    for e in (-130, -126, -125, -14, 0, 9, 100, 125):
        for f in (1.0, 1.0 + 2.0 ** -7, 1 - 2.0 ** -8):
            rows.append([6 * 2.0 ** e] + [t * f * 2.0 ** e for t in tie] + [-t * 2.0 ** e for t in tie])
        for top in (3.5, 3.515625, 6.96875, 7.0, 7.03125, 7.96875):
            rows.append([top * 2.0 ** e, -2.0 ** e, 0.0, -0.0, top * 2.0 ** e / 3])
    lim = torch.finfo(dtype)
    rows += [[lim.max, -lim.max / 2], [lim.tiny], [lim.smallest_normal / 8], [math.inf, 1.0],
             [1.0, -math.inf, 2.0], [math.nan], [0.0, -math.nan], [-0.0], []]
    x = torch.zeros(1, len(rows), 1, 64)
    for i, r in enumerate(rows):
        x[0, i, 0, :len(r)] = torch.tensor(r, dtype=torch.float64).float()
        x[0, i, 0, 33] = 1.0  # the second block has values of its own
    x = x.to(dtype)
    table, need = tables([len(rows)], 16)
    fill = torch.zeros(need, 1, 1, 544, dtype=torch.uint8)
    kc, vc = fill.to(device), fill.to(device)
    note(f"special {dtype}")
    write_kv_fp4(x.to(device), x.to(device), kc, vc, table.to(device), 0)
    assert torch.equal(kc.cpu(), storing(x, fill, table, [0], False))
    assert torch.equal(vc.cpu(), storing(x, fill, table, [0], True))
    k, v = read_kv_fp4(kc, vc, table.to(device), 0, len(rows), dtype=F32)
    want = torch.from_numpy(fp4.values(*fp4.quantise(x))).float()
    for got in (k, v):
        assert torch.equal(got.cpu().nan_to_num(nan=7e30), want.nan_to_num(nan=7e30))


def bound(dtype, D, n, scale, qn, kn, vmax):
    parts = {BF16: 1, F16: 2, F32: 3}[dtype]
    u = torch.finfo(dtype).eps / 2
    ds = (parts * D + 8) * 2.0 ** -24 * abs(scale) * qn * kn
    weights = 3 * u if dtype == BF16 else 2 * u + 2.0 ** -15 * (dtype == F16)
    return (4.04 * ds * math.exp(2 * ds) + weights + (n / 32 + 40) * 2.0 ** -23 + 2.0 ** -18) * vmax


class Batch:
    """Rows over a 4-bit cache. Whatever no row may see (spare pages, slots past a context) reads as
    NaN, both as elements and as scales."""

    def __init__(self, H, KVH, D, dtype, lens, q_len=1, bs=16, extra=0, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed + 7 * H + D + len(lens))
        self.lens, self.bs, self.dev = list(lens), bs, torch.device(device)
        self.table, need = tables(lens, bs, extra, seed)
        self.q = torch.randn(len(lens), q_len, H, D, generator=g).to(dtype)
        self.k, self.v = (fp4.values(*fp4.quantise(torch.randn(need, bs, KVH, D, generator=g)))
                          for _ in range(2))
        seen = np.zeros((need, bs), dtype=bool)
        for b, n in enumerate(lens):
            for pos in range(max(n, 0)):
                seen[int(self.table[b, pos // bs]), pos % bs] = True
        self.caches = []
        for x, is_values in ((self.k, False), (self.v, True)):
            codes, scale = fp4.quantise(torch.from_numpy(x))
            codes[~seen] = 15
            scale[~seen] = 255
            self.caches.append(fp4.pack(codes, scale, is_values).to(self.dev))

    def call(self, lens=None, **kw):
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.dev) if lens is None else lens
        return paged_attention_fp4(self.q.to(self.dev), *self.caches, self.table.to(self.dev), lens,
                                   **kw)

    def check(self, out, causal=True, window=None, scale=None, rows=None):
        B, T, H, D = self.q.shape
        scale = D ** -0.5 if scale is None else scale
        out = out.cpu().double()
        for b in range(B) if rows is None else rows:
            n = self.lens[b]
            if n <= 0:
                assert out[b].abs().max() == 0
                continue
            pages = self.table[b].numpy().copy()
            hole = (pages < 0) | (pages >= self.k.shape[0])
            pages[hole] = 0
            at = np.arange(n)
            k, v = (x[pages[at // self.bs], at % self.bs] for x in (self.k, self.v))
            live = ~hole[at // self.bs]
            keep = dense.keep_mask(n, T, causal, window) & live[None]
            want = torch.from_numpy(dense.attend_f64(self.q[b].double().numpy(), k, v, keep, scale))
            limit = bound(self.q.dtype, D, n, scale, self.q[b].double().norm(dim=-1).max().item(),
                          np.linalg.norm(k, axis=-1).max(), np.abs(v).max())
            err = (out[b] - want).abs().max().item()
            assert err <= limit, (b, n, err, limit)


# name -> (H, KVH, D, query type, lens, q_len, block size, causal, window)
CASES = {
    "one key": (8, 2, 64, BF16, [1], 1, 16, True, None),
    "around a tile": (8, 2, 128, BF16, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65], 1, 16, True, None),
    "around a tile, fp16": (14, 2, 64, F16, [0, 1, 15, 16, 17, 31, 32, 33, 64], 1, 16, True, None),
    "around a tile, fp32": (14, 2, 64, F32, [0, 1, 15, 16, 17, 31, 32, 33, 64], 1, 16, True, None),
    "ragged": (32, 8, 128, BF16, [700, 1, 333, 1025, 40, 0, 512], 1, 16, True, None),
    "ragged, fp16": (28, 4, 128, F16, [700, 1, 333, 1025, 40, 0, 512], 1, 16, True, None),
    "ragged, fp32": (28, 4, 128, F32, [700, 1, 333, 1025, 40, 0, 512], 1, 16, True, None),
    "no context": (4, 4, 64, BF16, [0, 0, -3], 1, 16, True, None),
    "32 dims": (16, 4, 32, BF16, [100, 33, 1], 1, 16, True, None),
    "96 dims": (24, 8, 96, BF16, [100, 33, 300], 1, 64, True, None),
    "96 dims, fp32": (24, 8, 96, F32, [100, 33, 300], 2, 32, True, None),
    "160 dims": (10, 2, 160, F16, [100, 133, 1], 1, 16, True, None),
    "192 dims": (6, 6, 192, BF16, [100, 133, 1], 3, 16, True, None),
    "224 dims": (9, 3, 224, F32, [90, 133], 1, 16, True, None),
    "256 dims": (8, 1, 256, BF16, [500, 77], 1, 16, True, None),
    "256 dims, 20 rows": (20, 1, 256, F32, [300, 77], 1, 48, True, None),
    "17 rows a head": (17, 1, 128, BF16, [400, 90], 1, 16, True, None),
    "33 rows a head": (33, 1, 64, BF16, [400, 90], 1, 16, True, None),
    "70 rows a head, fp16": (70, 1, 64, F16, [210, 90], 1, 16, True, None),
    "130 rows a head": (13, 1, 128, BF16, [400, 90, 7], 10, 16, True, None),
    "drafts": (28, 4, 128, F16, [200, 195, 410, 115, 3], 4, 16, True, None),
    "drafts longer than their context": (8, 4, 64, BF16, [3, 0, 40], 6, 16, True, None),
    "a prompt by itself": (14, 2, 64, BF16, [150, 150], 150, 16, True, None),
    "a prompt by itself, fp32": (4, 2, 96, F32, [130, 77], 77, 32, True, None),
    "a chunk": (28, 4, 128, BF16, [700, 333], 100, 16, True, None),
    "a chunk, fp16": (12, 4, 128, F16, [500, 133], 65, 16, True, None),
    "not causal": (8, 2, 128, BF16, [300, 20, 65], 9, 16, False, None),
    "not causal, fp32": (8, 2, 64, F32, [300, 20, 65], 40, 16, False, None),
    "window of one": (8, 2, 128, BF16, [300, 20, 1, 0], 1, 16, True, 1),
    "window inside a tile": (8, 2, 64, F16, [300, 20, 65, 7], 1, 16, True, 5),
    "window over drafts": (28, 4, 128, BF16, [300, 20, 465, 7], 4, 16, True, 33),
    "window over a chunk": (8, 2, 128, BF16, [400, 300], 90, 16, True, 40),
    "window, not causal": (8, 2, 64, F32, [200, 33], 20, 16, False, 9),
    "window past the context": (8, 2, 64, BF16, [200, 33], 2, 16, True, 1000),
    "pages of 48": (8, 2, 128, BF16, [340, 500, 145, 150], 2, 48, True, None),
    "pages of 256": (8, 2, 64, F16, [513, 600, 1000], 1, 256, True, None),
    "long": (4, 1, 128, BF16, [20000, 11000, 3], 1, 16, True, None),
    "long, fp32": (2, 1, 64, F32, [17700, 30001], 1, 64, True, None),
    "wide chunk, one a wave": (16, 2, 128, BF16, [700, 640], 600, 16, True, None),
    "wide chunk, 64 dims": (16, 8, 64, BF16, [300] * 4, 270, 16, True, None),
    "wide chunk, window": (16, 2, 128, BF16, [700, 90], 300, 32, True, 100),
    "wide chunk, not causal": (8, 2, 96, BF16, [333, 1000], 200, 16, False, None),
    "wide chunk, fp32": (16, 2, 128, F32, [500, 430], 400, 16, True, None),
    "wide chunk, 256 dims": (8, 1, 256, F16, [300, 170], 150, 16, True, None),
    "wide chunk, 256 dims, fp32": (8, 1, 256, F32, [300, 170], 150, 16, True, None),
    "wide chunk, 256 dims, one a wave": (8, 1, 256, BF16, [700, 640, 333, 610], 600, 16, True, None),
    "wide chunk, 256 dims, fp32, two a wave": (8, 1, 256, F32, [400, 340, 333, 377], 320, 16, False, 90),
    "wide chunk, fp16, one a wave": (16, 2, 128, F16, [700, 640], 600, 16, True, None),
    "two blocks of 16 rows": (28, 4, 128, BF16, [(i * 97) % 900 for i in range(30)], 4, 16, True, 300),
    "two blocks of 16 rows, fp32": (6, 2, 224, F32, [(i * 97) % 900 for i in range(30)], 7, 16, True, None),
    "drafts in a list": (28, 4, 128, BF16, [2500 - 37 * i for i in range(20)], 3, 16, True, None),
    "ragged in a list": (32, 8, 64, BF16, [1 + (i * 977) % 3100 for i in range(70)], 1, 16, True, None),
    "ragged in a list, fp32": (8, 4, 128, F32, [1 + (i * 977) % 3100 for i in range(30)], 1, 16, True, None),
    "ragged in a list, 256 dims": (4, 4, 256, F16, [1 + (i * 977) % 3100 for i in range(25)], 1, 16, True, None),
    "ragged in a list, window": (32, 8, 128, F16, [(i * 977) % 5100 for i in range(40)], 2, 16, True, 1500),
    "16 rows in a list": (16, 1, 64, BF16, [9000, 4000, 12000, 70, 0], 1, 16, True, None),
    "two row blocks in a list": (8, 2, 64, BF16, [9000, 3000, 5, 0], 10, 16, True, None),
    "row blocks in a list, fp32": (12, 2, 96, F32, [5000, 7100], 17, 32, True, None),
    "row blocks in a list, window": (8, 2, 128, BF16, [9000, 4100], 11, 16, True, 3500),
    "row blocks in a list, 192 dims": (8, 1, 192, F16, [6000, 4100], 9, 16, False, None),
    "more rows than a list takes": (1, 1, 64, BF16, [(i * 37) % 70 for i in range(2100)], 1, 16, True, None),
    "more rows than a list takes, drafts": (7, 1, 32, F16, [(i * 37) % 50 for i in range(2100)], 3, 16, True, None),
    "many rows": (8, 8, 64, BF16, [1 + (i * 37) % 150 for i in range(300)], 1, 16, True, None),
}


@pytest.mark.parametrize("name", list(CASES))
def test_against_64_bits(device, name):
    H, KVH, D, dtype, lens, q_len, bs, causal, window = CASES[name]
    x = Batch(H, KVH, D, dtype, lens, q_len, bs)
    note(f"attention {name}")
    x.check(x.call(causal=causal, window=window), causal, window)


@pytest.mark.parametrize("name", ["around a tile", "ragged", "ragged in a list", "ragged in a list, fp32",
                                  "ragged in a list, 256 dims", "many rows", "33 rows a head", "32 dims",
                                  "drafts in a list", "a chunk", "a chunk, fp16", "96 dims, fp32",
                                  "256 dims, 20 rows", "no context", "pages of 48"])
def test_short_contexts_under_wide_tables(device, name):
    """A table that could hold 40000 tokens: many short units in each share of a list, its plan in
    registers or LDS, and joins of units that several shares have."""
    H, KVH, D, dtype, lens, q_len, bs, causal, window = CASES[name]
    x = Batch(H, KVH, D, dtype, lens, q_len, bs, extra=40000 // bs)
    note(f"wide table {name}")
    x.check(x.call(causal=causal, window=window), causal, window)


@pytest.mark.parametrize("q_len", [1, 40])
def test_every_byte_it_reads_is_written(device, q_len):
    """A workspace of NaN past the header, which stays zero; twice: bit for bit the same."""
    x = Batch(32, 8, 128, BF16, [500, 480, 600, 481, 40] + [200 + 31 * i for i in range(9)], q_len)
    nbytes = nat.lib().msattn_fp4_workspace_bytes(14, q_len, 32, 8, 128, 600, nat.BF16)
    ws = torch.full((nbytes,), 255, dtype=torch.uint8, device=device)
    header = (64 + 4096) * 4
    ws[:header] = 0
    note(f"poisoned workspace {q_len}")
    a = x.call(workspace=ws, max_context=600)
    x.check(a)
    assert not ws[:header].any()
    ws[header:] = 255
    assert torch.equal(a, x.call(workspace=ws, max_context=600))


@pytest.mark.parametrize("KVH,q_len", [(1, 1), (2, 4), (8, 1), (20, 1), (40, 3)])
def test_partials_are_written_before_they_are_read(device, KVH, q_len):
    """The same where units are cut: parts of few units, among them ones of no key, of one and of
    fewer groups than parts, and a list's shares."""
    lens = [0, 1, 40, 257, 300, 900, 9000, 2300]
    x = Batch(KVH, KVH, 64, F16, lens, q_len, extra=1500)
    nbytes = nat.lib().msattn_fp4_workspace_bytes(8, q_len, KVH, KVH, 64, 30000, nat.F16)
    ws = torch.full((nbytes,), 255, dtype=torch.uint8, device=device)
    header = (64 + 4096) * 4
    ws[:header] = 0
    note(f"poisoned partials {KVH} {q_len}")
    a = x.call(workspace=ws, max_context=30000)
    x.check(a)
    assert not ws[:header].any()
    ws[header:] = 255
    assert torch.equal(a, x.call(workspace=ws, max_context=30000))


@pytest.mark.parametrize("q_len", [1, 3, 50])
def test_holes_are_not_read(device, q_len):
    x = Batch(8, 2, 128, BF16, [300, 250, 193, 200, 90], q_len)
    x.table[0, 4], x.table[1, 15], x.table[3, 0], x.table[4, 5] = -1, x.k.shape[0], -7, 2 ** 31 - 1
    x.table[2, :] = -1
    note(f"holes {q_len}")
    x.check(x.call())


def test_a_larger_table_and_a_bound_on_the_context(device):
    x = Batch(14, 2, 64, F16, [140, 129, 200, 333], 1, extra=40)
    note("max_context")
    want = x.call()
    x.check(want)
    wide = torch.tensor(x.lens, dtype=torch.int64, device=device)
    assert torch.equal(want, x.call(lens=wide))
    wide[2] += 2 ** 32  # past any table: as many keys as max_context
    x.check(x.call(lens=wide, max_context=200), rows=[0, 1, 2])
    x.check(x.call(lens=x.lens))  # (host lengths: the bound is their largest)
    full = torch.tensor(x.lens, dtype=torch.int32, device=device)
    x.lens = [min(n, 150) for n in x.lens]
    x.check(x.call(lens=full, max_context=150))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scales(device, scale):
    x = Batch(8, 2, 64, F16, [120, 100, 97], 2)
    note(f"scale {scale}")
    x.check(x.call(scale=scale), scale=scale)


@pytest.mark.parametrize("q_len,D", [(1, 128), (5, 64), (40, 128), (3, 256)])
def test_nan_reaches_the_queries_that_see_it(device, q_len, D):
    """A NaN block of a value: those 32 dims of the queries that see its key. Of a key: all of them."""
    lens = [70, 45]
    for which in (0, 1):
        x = Batch(8, 2, D, BF16, lens, q_len)
        clean = x.call()
        for b, key, block in ((0, lens[0] - 2, 1), (1, 7, 0)):
            page, slot = int(x.table[b, key // 16]), key % 16
            x.caches[which][page, 1, 0, 8 * D + 16 * block + slot] = 255  # KV head 1: heads 4 .. 7
        note(f"nan {which} {q_len} {D}")
        out = x.call()
        for b, key, block in ((0, lens[0] - 2, 1), (1, 7, 0)):
            for t in range(q_len):
                sees = key <= lens[b] - q_len + t
                hit = torch.zeros(8, D, dtype=torch.bool)
                if sees:
                    hit[4:, 32 * block:32 * block + 32] = True
                    if which == 0:
                        hit[4:] = True
                got = out[b, t].cpu()
                assert torch.equal(got.isnan(), hit), (which, b, t)
                # (a key's NaN may move the running maximum of rows it shares a wave with)
                near = (got.float() - clean[b, t].cpu().float()).abs()
                assert near[~hit].max() <= 2.0 ** -7 * clean.float().abs().max().item() \
                    if (~hit).any() else True


def test_infinite_queries(device):
    x = Batch(4, 2, 64, F32, [40, 50], 1)
    x.q[0, 0, 1, 3] = math.inf
    x.q[1, 0, 2, 5] = math.nan
    note("infinite query")
    out = x.call().cpu()
    assert not out[0, 0, 0].isnan().any() and not out[0, 0, 2:].isnan().any()
    assert out[1, 0, 2].isnan().all() and not out[1, 0, :2].isnan().any()
    s = torch.from_numpy(x.k[x.table[0].long()].reshape(-1, 2, 64)[:40, 0]) @ x.q[0, 0, 1].double()
    assert out[0, 0, 1].isnan().all() == bool(s.isnan().any() or (s == math.inf).any())


def test_through_the_class_in_a_run(device):
    """A prompt in two chunks, then decoded tokens, through PagedAttention: every step against 64
    bits over what the cache holds, and the reads against the oracle's quantisation."""
    H, KVH, D, bs, lens = 8, 2, 64, 32, [75, 40]
    pa = PagedAttention(H, KVH, D, num_blocks=12, block_size=bs, dtype=BF16, device=device,
                        kv_dtype=torch.float4_e2m1fn_x2)
    kc, vc = pa.allocate_kv_cache()
    table, _ = tables([90, 90], bs, seed=4)
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(2, 90, KVH, D, generator=g).to(BF16) for _ in range(2))
    stored = [fp4.values(*fp4.quantise(x)) for x in (k, v)]
    dev_table = table.to(device)
    at = [0, 0]
    for step in (30, 37, 1, 1, 1):
        q = torch.randn(2, step, H, D, generator=g).to(BF16)
        new = [torch.stack([x[b, at[b]:at[b] + step] for b in range(2)]).to(device) for x in (k, v)]
        pa.write_kv(kc, vc, *new, dev_table, torch.tensor(at, dtype=torch.int32, device=device))
        at = [a + step for a in at]
        note(f"run, {at}")
        out = pa(q.to(device), kc, vc, dev_table, at).cpu().double()
        for b in range(2):
            kb, vb = (x[b, :at[b]] for x in stored)
            want = torch.from_numpy(dense.attend_f64(
                q[b].double().numpy(), kb, vb, dense.keep_mask(at[b], step, True, None), D ** -0.5))
            limit = bound(BF16, D, at[b], D ** -0.5, q[b].double().norm(dim=-1).max().item(),
                          np.linalg.norm(kb, axis=-1).max(), np.abs(vb).max())
            assert (out[b] - want).abs().max().item() <= limit
        for got, want in zip(read_kv_fp4(kc, vc, dev_table, 0, at[0], dtype=F32), stored):
            assert torch.equal(got.cpu().double(), torch.from_numpy(want[:, :at[0]]))
    with pytest.raises(ValueError, match="4-bit"):
        pa(q.to(device), kc, vc, dev_table, at, backend="triton_flash")


def test_captured_and_replayed(device):
    """Write and attention in one graph, replayed over changing inputs, lengths and tables; a
    second graph with a workspace of its own in between."""
    H, KVH, D = 14, 2, 64
    x = Batch(H, KVH, D, BF16, [100, 1, 333, 64], 1)
    table, q = x.table.to(device), x.q.to(device)
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device)
    new = torch.randn(2, 4, 1, KVH, D, device=device, generator=torch.Generator(device).manual_seed(1)).to(BF16)
    kc, vc = x.caches

    def step():
        write_kv_fp4(new[0], new[1], kc, vc, table, lens - 1)
        return paged_attention_fp4(q, kc, vc, table, lens, max_context=400)

    side = torch.cuda.Stream(device)
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    note("capture")
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for i in range(4):
        q.normal_()
        new.normal_()
        lens.copy_(torch.tensor([[100, 1, 333, 64], [99, 0, 320, 33], [17, 1, 250, 0]][i % 3]))
        note(f"replay {i}")
        for gr, out in graphs:
            gr.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, step())


def test_graphed_runner(device):
    """Bucketed graphs over 4-bit caches: three layers, padded buckets, against eager steps."""
    H, KVH, D, bs, L = 8, 2, 64, 16, 3
    g = torch.Generator(device).manual_seed(3)

    def layers():
        out = []
        for _ in range(L):
            pa = PagedAttention(H, KVH, D, num_blocks=24, block_size=bs, dtype=BF16, device=device,
                                kv_dtype=torch.float4_e2m1fn_x2)
            out.append(DecodeLayer(pa, *pa.allocate_kv_cache()))
        return out

    pair = [GraphedDecodeRunner(layers(), 6, buckets=(1, 2, 4), dtype=BF16) for _ in range(2)]
    assert (pair[0].block_size, pair[0].num_kv_heads, pair[0].head_dim) == (bs, KVH, D)
    tables_ = [[0, 5, 9], [1, 2], [3, 4, 6, 7], [8]]
    for step, (rows, ctx) in enumerate([((0, 1, 2), [0, 0, 0]), ((0, 1, 2, 3), [1, 1, 1, 0]),
                                        ((2,), [2]), ((0, 1, 2), [2, 2, 3]), ((3, 0), [1, 3])]):
        B = len(rows)
        q = torch.randn(L, B, 1, H, D, device=device, generator=g).to(BF16)
        k, v = (torch.randn(L, B, 1, KVH, D, device=device, generator=g).to(BF16) for _ in range(2))
        note(f"runner step {step}")
        a, b = (r.decode(q, k, v, [tables_[i] for i in rows], ctx, use_graph=use)
                for r, use in zip(pair, (True, False)))
        torch.cuda.synchronize()
        assert torch.equal(a, b)
        for x, y in zip(pair[0].layers, pair[1].layers):
            assert torch.equal(x.k_cache, y.k_cache) and torch.equal(x.v_cache, y.v_cache)
        if ctx[0] == 0:  # one key: its value, as stored
            want = fp4.values(*fp4.quantise(v[:, 0].cpu()))
            got = a[:, 0].cpu().double().reshape(L, 1, KVH, H // KVH, D)
            assert np.array_equal(got.numpy(), np.broadcast_to(want[:, :, :, None], got.shape))
    with pytest.raises(ValueError, match="no rope"):
        GraphedDecodeRunner(layers(), 6, dtype=BF16, rope=(torch.ones(9, D), torch.zeros(9, D)))


def test_on_another_stream(device):
    x = Batch(8, 2, 128, BF16, [300, 120], 1)
    want = x.call()
    side = torch.cuda.Stream(device)
    note("side stream")
    with torch.cuda.stream(side):
        got = x.call()
    side.synchronize()
    assert torch.equal(got, want)


def test_two_streams_and_graphs_at_once(device):
    """Shares and joins of four calls that run together, eager ones and replayed ones, each with its
    stream's or graph's workspace; 16-bit calls on the same workspace in between."""
    x = Batch(8, 2, 64, BF16, [9000, 3000, 700, 12000], 1)
    table, q = x.table.to(device), x.q.to(device)
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device)
    want = x.call()
    x.check(want)
    pa = PagedAttention(8, 2, 64, num_blocks=64, block_size=16, dtype=BF16, device=device)
    kc, vc = (torch.randn(t.shape, device=device, generator=torch.Generator(device).manual_seed(3))
              .to(BF16) for t in pa.allocate_kv_cache())
    table16 = torch.arange(64, dtype=torch.int32, device=device).view(1, 64)
    want16 = pa(q[:1], kc, vc, table16, [1000])
    streams = [torch.cuda.Stream(device) for _ in range(2)]
    graphs = []
    note("capture")
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(device))
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = paged_attention_fp4(q, *x.caches, table, lens)
        graphs.append((gr, out))
    torch.cuda.synchronize()
    for i in range(3):
        note(f"together {i}")
        outs = []
        for s, (gr, out) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(4):
                    outs.append(paged_attention_fp4(q, *x.caches, table, lens))
                    gr.replay()
                    got16 = pa(q[:1], kc, vc, table16, [1000])
                outs += [out, outs[-1]]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        assert torch.equal(got16, want16)
        for _, out in graphs:
            out.zero_()
        torch.cuda.synchronize()


def test_caches_past_4_gib(device):
    """Pages 2^29 bytes apart: written, read and attended over as the same pages side by side."""
    x = Batch(8, 2, 64, BF16, [70, 33], 1)
    nb = x.caches[0].shape[0]
    kc, vc = (c.new_empty((nb - 1) * 2 ** 29 + 8 * 4096).as_strided(c.shape, (2 ** 29, 4096, 544, 1))
              for c in x.caches)
    kc.copy_(x.caches[0])
    vc.copy_(x.caches[1])
    g = torch.Generator().manual_seed(9)
    new = [torch.randn(2, 12, 2, 64, generator=g).to(BF16).to(device) for _ in range(2)]
    table, start = x.table.to(device), [n - 12 for n in x.lens]
    note("far pages")
    for caches in ((kc, vc), x.caches):
        write_kv_fp4(*new, *caches, table, start)
    assert torch.equal(kc, x.caches[0]) and torch.equal(vc, x.caches[1])
    for a, b in zip(read_kv_fp4(kc, vc, table, 0, 70), read_kv_fp4(*x.caches, table, 0, 70)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device)
    want = x.call()
    assert torch.equal(paged_attention_fp4(x.q.to(device), kc, vc, table, lens), want)


def test_shared_and_expanded_inputs(device):
    """One tensor as keys and values, heads and tokens of one row by stride 0, one query for all
    rows, and k inside the cache's own memory."""
    x = Batch(8, 2, 64, BF16, [64, 64, 64], 1)
    table = x.table.to(device)
    row = torch.randn(3, 1, 1, 64, device=device, generator=torch.Generator(device).manual_seed(1)).to(BF16)
    fresh = [torch.zeros_like(c) for c in x.caches]
    note("expanded")
    wide = row.expand(3, 20, 2, 64)
    write_kv_fp4(wide, wide, *x.caches, table, 7)
    write_kv_fp4(wide.contiguous(), wide.clone(), *fresh, table, 7)
    k, v = read_kv_fp4(*x.caches, table, 7, 20)
    assert torch.equal(k, v) and all(torch.equal(a, b) for a, b in
                                     zip((k, v), read_kv_fp4(*fresh, table, 7, 20)))
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device)
    q = x.q[:1].to(device)
    assert torch.equal(paged_attention_fp4(q.expand(3, 1, 8, 64), *x.caches, table, lens),
                       paged_attention_fp4(q.repeat(3, 1, 1, 1), *x.caches, table, lens))
    # the last pages of the caches, which no table names, as the keys' and values' memory
    pool = torch.zeros(2, 8, 2, 1, 544, dtype=torch.uint8, device=device)
    kc, vc = pool.unbind(0)
    own = [c[6].view(-1)[:512].view(BF16).view(1, 2, 2, 64) for c in (kc, vc)]
    for t in own:
        t.normal_()
    kept = [t.clone() for t in own]
    one = torch.zeros(1, 2, dtype=torch.int32, device=device)
    write_kv_fp4(*own, kc, vc, one, 3)
    want = allocate_fp4_cache(8, 16, 2, 64, device=device)
    write_kv_fp4(*kept, *want, one, 3)
    assert torch.equal(kc[0], want[0][0]) and torch.equal(vc[0], want[1][0])
    assert all(torch.equal(a, b) for a, b in zip(own, kept))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_parts_of_tiles_read_back(device, dtype):
    """Every start in a tile and every number of tokens up to two tiles: what lies beside the answer
    in its buffer is the next row's."""
    KVH, D = 2, 96
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, 64, KVH, D, generator=g).to(BF16).to(device)
    kc, vc = allocate_fp4_cache(5, 16, KVH, D, device=device)
    table = torch.tensor([[3, 1, 4, 0]], dtype=torch.int32, device=device)
    write_kv_fp4(x, -x, kc, vc, table)
    k, v = read_kv_fp4(kc, vc, table, 0, 64, dtype=dtype)
    two = table.expand(16, 4)
    starts = torch.arange(16, dtype=torch.int32, device=device)
    note(f"parts {dtype}")
    for n in (1, 2, 3, 15, 16, 17, 31, 32, 33):
        a, b = read_kv_fp4(kc, vc, two, starts, n, dtype=dtype)
        for i in range(16):
            assert torch.equal(a[i], k[0, i:i + n]) and torch.equal(b[i], v[0, i:i + n])


def test_views_outputs_and_pages_apart(device):
    """A strided query is read in place, a cache of one pool's layers, the output over the query."""
    x = Batch(8, 2, 128, F16, [300, 120], 3)
    want = x.call()
    qkv = torch.empty(2, 3, 12, 128, dtype=F16, device=device)
    qkv[:, :, 2:10] = x.q.to(device)
    lens = torch.tensor(x.lens, device=device)
    table = x.table.to(device).long()
    note("views")
    assert torch.equal(paged_attention_fp4(qkv[:, :, 2:10], *x.caches, table, lens), want)
    flat = torch.empty(2 * 3 * 8 * 128 + 3, dtype=F16, device=device)[3:].view(2, 3, 8, 128)
    flat.copy_(x.q)
    assert torch.equal(paged_attention_fp4(flat, *x.caches, table, lens), want)
    nb = x.caches[0].shape[0]
    pool = torch.zeros(nb, 5, 2, 1, 1088, dtype=torch.uint8, device=device)
    pool[:, 1], pool[:, 3] = x.caches[0], x.caches[1]
    assert torch.equal(paged_attention_fp4(x.q.to(device), pool[:, 1], pool[:, 3], table, lens), want)
    q = x.q.to(device)
    assert torch.equal(paged_attention_fp4(q, *x.caches, table, lens, out=q), want)
    assert torch.equal(q, want)


def test_refusals(device):
    kc, vc = allocate_fp4_cache(8, 16, 2, 64, device=device)
    table = torch.zeros(2, 3, dtype=torch.int32, device=device)
    x = torch.zeros(2, 1, 2, 64, device=device)
    q = torch.zeros(2, 1, 4, 64, device=device)
    with pytest.raises(ValueError, match="do not match"):
        write_kv_fp4(x[:, :, :1], x[:, :, :1], kc, vc, table)
    with pytest.raises(ValueError, match="do not match"):
        write_kv_fp4(x[..., :32], x[..., :32], kc, vc, table)
    with pytest.raises(ValueError, match="must both be"):
        write_kv_fp4(x, x[:1], kc, vc, table)
    with pytest.raises(ValueError, match="share a dtype"):
        write_kv_fp4(x, x.half(), kc, vc, table)
    with pytest.raises(ValueError, match="unsupported dtype"):
        write_kv_fp4(x.double(), x.double(), kc, vc, table)
    with pytest.raises(ValueError, match="fewer rows"):
        write_kv_fp4(x, x, kc, vc, table[:1])
    with pytest.raises(ValueError, match="one entry per batch row"):
        write_kv_fp4(x, x, kc, vc, table, [1])
    with pytest.raises(ValueError, match="uint8"):
        write_kv_fp4(x, x, kc.view(torch.int8), vc.view(torch.int8), table)
    with pytest.raises(ValueError, match="share a uint8"):
        write_kv_fp4(x, x, kc, vc[:4], table)
    with pytest.raises(ValueError, match="tile of"):
        write_kv_fp4(x, x, kc[..., :540], vc[..., :540], table)
    with pytest.raises(ValueError, match="unsupported dtype"):
        read_kv_fp4(kc, vc, table, 0, 4, dtype=torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="negative"):
        read_kv_fp4(kc, vc, table, 0, -1)
    with pytest.raises(ValueError, match="head_dim mismatch"):
        paged_attention_fp4(q[..., :32], kc, vc, table, [1, 1])
    with pytest.raises(ValueError, match="multiple of num_kv_heads"):
        paged_attention_fp4(q[:, :, :3], kc, vc, table, [1, 1])
    with pytest.raises(ValueError, match="window"):
        paged_attention_fp4(q, kc, vc, table, [1, 1], window=0)
    with pytest.raises(ValueError, match="rows for a batch"):
        paged_attention_fp4(q, kc, vc, table[:1], [1, 1])
    with pytest.raises(ValueError, match="exceeds"):
        paged_attention_fp4(q, kc, vc, table, [1, 49])
    with pytest.raises(ValueError, match="out must"):
        paged_attention_fp4(q, kc, vc, table, [1, 1], out=q.half())
    with pytest.raises(ValueError, match="unsupported dtype"):
        paged_attention_fp4(q.double(), kc, vc, table, [1, 1])
    assert paged_attention_fp4(q[:, :0], kc, vc, table, [1, 1]).shape == (2, 0, 4, 64)
    write_kv_fp4(x[:, :0], x[:, :0], kc, vc, table)
