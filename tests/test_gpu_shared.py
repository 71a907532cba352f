"""Attention behind several shared prefixes (paged_attention_shared) on the GPU, against 64 bits.

Tolerance. Scores are fp32 sums of exact products: off by at most |ds| = (D + 8) 2^-24 scale |q||k|
(products, D additions, the scale), so a weight is off by a factor e^(2 |ds|); it is rounded to the
query type (u = eps / 2 relative; fp16 weights below 2^-14 by 2^-25 absolute, beside a largest
weight of 1 or more), in the numerator and in the sum alike, and the output is rounded once more. Outputs
are weighted means of V: the whole is at most (4.04 |ds| e^(2 |ds|) + 3 u + n 2^-24 [fp16] + 2^-18)
max |V| over the n visible keys, the last term for the hardware's 2^x and the joins in fp32.
"""
import math
import random

import pytest
import torch

from miniserve_amd import PagedAttention, _native as nat, paged_attention, paged_attention_shared
from oracle import dense

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn


def note(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


class Batch:
    """Rows in groups: `groups` = [(first row, rows, prefix pages)], lens per row. Whatever no row
    may see (unused pages, slots past every context that holds the page) is NaN."""

    def __init__(self, H, KVH, D, qt, kt, groups, lens, q_len=1, bs=16, extra=0, seed=0,
                 device="cuda"):
        g = torch.Generator().manual_seed(seed + 7 * H + D + len(lens))
        self.B, self.bs, self.q_len, self.lens = len(lens), bs, q_len, list(lens)
        W = max(1, max([-(-n // bs) for n in lens] + [p for _, _, p in groups])) + extra
        self.rows = [groups[0][0]] if groups else []
        self.pages = []
        for r0, n, p in groups:
            assert r0 == self.rows[-1]
            self.rows.append(r0 + n)
            self.pages.append(p)
        need = sum(self.pages) + self.B * W + 2
        perm = torch.randperm(need, generator=g).tolist()
        table = torch.full((self.B, W), -1, dtype=torch.int32)
        seen = {}
        first = [0] * self.B
        for (r0, n, p) in groups:
            ids = [perm.pop() for _ in range(p)]
            for b in range(r0, r0 + n):
                table[b, :p] = torch.tensor(ids, dtype=torch.int32)
                first[b] = p
        for b in range(self.B):
            for c in range(first[b], -(-lens[b] // bs)):
                table[b, c] = perm.pop()
            for c in range(W):
                if table[b, c] >= 0:
                    page = int(table[b, c])
                    seen[page] = max(seen.get(page, 0), min(bs, max(0, lens[b] - c * bs)))
        x = [torch.randn(need, bs, KVH, D, generator=g) for _ in range(2)]
        for page in range(need):
            for t in x:
                t[page, seen.get(page, 0):] = math.nan
        self.kc, self.vc = (t.to(kt) for t in x)
        self.table = table
        self.q = torch.randn(self.B, q_len, H, D, generator=g).to(qt)
        self.dev = torch.device(device)

    def call(self, fn=paged_attention_shared, lens=None, **kw):
        args = [t.to(self.dev) for t in (self.q, self.kc, self.vc, self.table)]
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.dev) if lens is None else lens
        if fn is paged_attention_shared:
            return fn(*args, lens, self.rows, self.pages, **kw)
        return fn(*args, lens, **kw)

    def check(self, out, rows=None, scale=None):
        B, T, H, D = self.q.shape
        KVH = self.kc.shape[2]
        scale = D ** -0.5 if scale is None else scale
        u = torch.finfo(self.q.dtype).eps / 2
        out = out.cpu().double()
        for b in range(B) if rows is None else rows:
            n = self.lens[b]
            if n <= 0:
                assert out[b].abs().max() == 0
                continue
            pages = self.table[b].clone()
            hole = (pages < 0) | (pages >= self.kc.shape[0])
            pages[hole] = 0
            k = torch.from_numpy(dense.gather_rows(self.kc, pages, n, self.q.dtype))
            v = torch.from_numpy(dense.gather_rows(self.vc, pages, n, self.q.dtype))
            keep = torch.from_numpy(dense.keep_mask(n, T, True, None))
            live = ~hole[torch.arange(n) // self.bs]
            keep &= live[None]
            k[~live], v[~live] = 0, 0
            assert bool(k.isfinite().all()), "the test's own pages"
            want = torch.from_numpy(dense.attend_f64(self.q[b].double().numpy(), k.numpy(),
                                                     v.numpy(), keep.numpy(), scale))
            ds = (D + 8) * 2.0 ** -24 * abs(scale) * \
                (self.q[b].double().norm(dim=-1).max() * k.norm(dim=-1).max()).item()
            bound = (4.04 * ds * math.exp(2 * ds) + 3 * u + 2.0 ** -18 +
                     (n * 2.0 ** -24 if self.q.dtype == F16 else 0)) * v.abs().max().item()
            err = (out[b] - want).abs().max().item()
            assert err <= bound, (b, n, err, bound)


# name -> (H, KVH, D, query, cache, groups, lens, q_len, block size)
CASES = {
    "two rows, one page": (14, 2, 64, BF16, BF16, [(0, 2, 1)], [17, 30], 1, 16),
    "ragged groups, loose rows around": (
        32, 8, 128, BF16, BF16, [(1, 3, 9), (4, 2, 40), (6, 4, 3)],
        [77, 200, 145, 500, 641, 1300, 49, 100, 70, 48, 333, 5], 1, 16),
    "empty and single-row groups": (
        8, 2, 128, F16, F16, [(0, 0, 4), (0, 1, 5), (1, 0, 2), (1, 3, 8), (4, 0, 1)],
        [100, 129, 128, 300, 60], 1, 16),
    "contexts that end in the prefix": (
        16, 4, 64, F16, F16, [(0, 7, 20)], [0, 1, 150, 319, 320, 321, 700], 1, 16),
    "no context at all": (4, 4, 64, BF16, BF16, [(0, 3, 2)], [0, 0, 0], 1, 16),
    "only prefixes": (28, 4, 128, BF16, BF16, [(0, 4, 17)], [272, 272, 272, 272], 1, 16),
    "no shared page": (28, 4, 128, BF16, BF16, [(0, 2, 0), (2, 2, 0)], [30, 270, 129, 1], 1, 16),
    "drafts of three": (28, 4, 128, F16, F16, [(0, 3, 12), (3, 2, 7)],
                        [200, 195, 410, 115, 300], 3, 16),
    "drafts that begin in the prefix": (8, 4, 64, BF16, BF16, [(0, 4, 10)],
                                        [163, 160, 165, 400], 5, 16),
    "drafts longer than their context": (8, 4, 64, BF16, BF16, [(0, 3, 2)], [3, 0, 40], 6, 16),
    "33 rows a unit": (11, 1, 128, F16, F16, [(0, 3, 30)], [500, 490, 700], 1, 16),
    "65 rows a unit": (13, 1, 64, BF16, BF16, [(0, 5, 21)], [400, 350, 337, 500, 336], 1, 16),
    "129 rows, two blocks": (43, 1, 128, BF16, BF16, [(0, 3, 25)], [500, 480, 401], 1, 16),
    "300 rows, three blocks": (30, 1, 64, F16, F16, [(0, 10, 14)], [230 + 9 * i for i in range(10)], 1, 16),
    "96 query rows a batch row": (24, 1, 64, BF16, BF16, [(0, 2, 9)], [160, 250], 4, 16),
    "pages of 32": (14, 2, 64, BF16, BF16, [(0, 3, 5)], [161, 250, 200], 1, 32),
    "pages of 48": (8, 2, 128, BF16, BF16, [(0, 2, 7), (2, 2, 3)], [340, 500, 145, 150], 2, 48),
    "pages of 256": (8, 2, 128, BF16, BF16, [(0, 3, 2)], [513, 600, 1000], 1, 256),
    "fp8, 16 rows": (32, 8, 128, BF16, FP8, [(0, 4, 33)], [600, 529, 700, 900], 1, 16),
    "fp8, 64 dims": (16, 2, 64, F16, FP8, [(0, 3, 20), (3, 3, 9)], [340, 400, 321, 150, 145, 290], 1, 16),
    "fp8, drafts": (28, 4, 128, F16, FP8, [(0, 6, 11)], [180, 200, 333, 181, 179, 410], 4, 16),
    "fp8, 200 rows": (40, 1, 64, BF16, FP8, [(0, 5, 40)], [650, 700, 800, 641, 660], 1, 16),
    "one KV head, long": (4, 1, 128, BF16, BF16, [(0, 3, 600)], [9700, 11000, 20000], 1, 16),
    "one KV head, long, 64 dims": (2, 1, 64, F16, F16, [(0, 2, 1100)], [17700, 30001], 1, 16),
    "fp8, long": (4, 1, 128, F16, FP8, [(0, 2, 600)], [9700, 19001], 1, 16),
    "many short rows": (8, 8, 64, BF16, BF16, [(20 * i, 20, 2 + i) for i in range(6)],
                        [(2 + i // 20) * 16 + 1 + (i * 37) % 150 for i in range(120)], 1, 16),
}


@pytest.mark.parametrize("name", list(CASES))
def test_against_64_bits(device, name):
    H, KVH, D, qt, kt, groups, lens, q_len, bs = CASES[name]
    x = Batch(H, KVH, D, qt, kt, groups, lens, q_len, bs)
    note(f"shared {name}")
    x.check(x.call())


@pytest.mark.parametrize("kt", [BF16, FP8])
def test_every_byte_it_reads_is_written(device, kt):
    """A workspace full of NaN past the header, which stays as it is; twice: bit for bit the same."""
    x = Batch(32, 8, 128, BF16, kt, [(0, 5, 30), (5, 9, 12)],
              [500, 480, 600, 481, 490] + [200 + 31 * i for i in range(9)] + [77], 1)
    ws = torch.full((nat.lib().msattn_shared_workspace_bytes(15, 1, 32, 8, 128, 600, 2),), 255,
                    dtype=torch.uint8, device=device)
    header = (64 + 4096) * 4
    ws[:header] = 0
    note(f"poisoned workspace {kt}")
    a = x.call(workspace=ws, max_context=600)
    x.check(a)
    assert not ws[:header].any()
    ws[header:] = 255
    assert torch.equal(a, x.call(workspace=ws, max_context=600))


def test_holes_are_not_read(device):
    x = Batch(8, 2, 128, BF16, BF16, [(0, 3, 12), (3, 2, 5)], [300, 250, 193, 200, 90], 2)
    for b in range(3):
        x.table[b, 4] = -1      # a hole in the first group's prefix
    x.table[0, 14], x.table[1, 15], x.table[4, 5] = -7, x.kc.shape[0], 2 ** 31 - 1
    note("holes")
    x.check(x.call())
    # a row of holes alone
    x.table[2, :] = -1
    x.rows, x.pages = [3, 5], [5]
    x.check(x.call())


def test_a_larger_table_and_a_bound_on_the_context(device):
    x = Batch(14, 2, 64, F16, F16, [(0, 4, 8)], [140, 129, 200, 333], 1, extra=40)
    note("max_context")
    want = x.call()
    x.check(want)
    assert torch.equal(want, x.call(lens=x.lens))  # (host lengths: the bound is their largest)
    x.lens = [min(n, 150) for n in x.lens]
    long = torch.tensor([140, 129, 200, 333], dtype=torch.int32, device=device)
    x.check(x.call(lens=long, max_context=150))


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scales(device, scale):
    x = Batch(8, 2, 64, F16, F16, [(0, 3, 6)], [120, 100, 97], 2)
    note(f"scale {scale}")
    x.check(x.call(scale=scale), scale=scale)


def test_strided_caches(device):
    """Padded pools, heads before slots, and offsets past 32 bits."""
    x = Batch(8, 2, 64, BF16, BF16, [(0, 3, 9)], [200, 150, 145], 1)
    want = x.call()
    x.check(want)
    rows, pages = x.rows, x.pages
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device)
    tab, q = x.table.to(device), x.q.to(device)
    def padded(t):
        b = torch.full((*t.shape[:3], 72), math.nan, dtype=t.dtype, device=device)
        b[..., :64] = t.to(device)
        return b[..., :64]
    def by_head(t):
        return t.to(device).transpose(1, 2).contiguous().transpose(1, 2)
    for form in (padded, by_head):
        note(form.__name__)
        assert torch.equal(want, paged_attention_shared(q, form(x.kc), form(x.vc), tab, lens, rows, pages))
    note("offsets past 32 bits")
    nb = 2 ** 31 // (16 * 8 * 128) + 60
    y = Batch(16, 8, 128, F16, FP8, [(0, 3, 9)], [200, 150, 145], 1)
    big = [torch.zeros(nb, 16, 8, 128, dtype=torch.uint8, device=device) for _ in range(2)]
    base = nb - y.kc.shape[0]
    for b, t in zip(big, (y.kc, y.vc)):
        b[base:] = t.view(torch.uint8).to(device)
    tab = torch.where(y.table >= 0, y.table + base, y.table).to(device)
    out = paged_attention_shared(y.q.to(device), big[0].view(FP8), big[1].view(FP8), tab, lens,
                                 y.rows, y.pages)
    y.check(out)


def test_infinities_and_nan(device):
    """NaN and infinities where no key is visible leave no trace (every test's pages hold NaN
    there); a NaN key or query makes its rows NaN, an infinite value its rows infinite."""
    x = Batch(4, 2, 64, BF16, BF16, [(0, 2, 4), (2, 2, 4)], [100, 90, 80, 120], 1)
    x.kc[x.table[0, 1], 3, 0] = math.nan      # a prefix key of rows 0 and 1, KV head 0
    x.vc[x.table[2, 5 - 1], 2, 1, 7] = math.inf  # an own value of row 2, KV head 1
    x.q[3, 0, 1] = math.nan
    note("NaN and infinities")
    out = x.call().float().cpu()
    nan = out.isnan()
    assert bool(nan[:2, :, :2].all()) and not bool(nan[:2, :, 2:].any())
    assert bool((out[2, 0, 2:, 7] == math.inf).all()) and int(out.isinf().sum()) == 2
    assert bool(nan[3, 0, 1].all()) and not bool(nan[3, 0, [0, 2, 3]].any())


@pytest.mark.parametrize("q_len,short", [(1, 40), (1, 63), (3, 65), (3, 40), (4, 2)])
def test_rows_that_do_not_see_the_whole_prefix(device, q_len, short):
    """A key and a value of NaN and an infinite one where only the other rows of the group see them
    leave no trace in the short row, which is as exact as ever."""
    x = Batch(4, 2, 128, BF16, BF16, [(0, 4, 4)], [100, short, 80, 120], q_len)
    clean = x.call().float().cpu()
    x.check(clean)
    # positions that none of the short row's queries but its last may see
    for pos, t, bad in ((max(short, 50), x.vc, math.nan), (max(short, 51), x.vc, math.inf),
                        (max(short, 52), x.kc, math.nan)):
        if pos < 64:
            t[x.table[0, pos // 16], pos % 16] = bad
    note(f"short row {short}, {q_len} queries")
    out = x.call().float().cpu()
    assert torch.equal(out[1], clean[1])
    if short < 64:
        assert bool(out[[0, 2, 3]].isnan().all())


@pytest.mark.parametrize("gone", [[0], [0, 1], [2], [0, 1, 2, 3]])
def test_padding_rows_in_a_group(device, gone):
    """Rows of a group that hold no sequence (length 0, an empty table), its first among them."""
    lens = [0 if b in gone else n for b, n in enumerate([100, 90, 80, 120])] + [70, 66]
    x = Batch(8, 2, 64, BF16, BF16, [(0, 4, 4), (4, 2, 2)], lens, 1)
    for b in gone:
        x.table[b] = -1
    note(f"rows {gone} empty")
    x.check(x.call())


@pytest.mark.parametrize("seed", range(32))
def test_fuzz(device, seed):
    """Seeded shapes: loose rows before, between and after groups, groups of one and of many, empty
    and short rows, prefixes of no page, contexts ending on and off tiles, up to 64 query rows."""
    r = random.Random(7000 + seed)
    KVH, G = r.choice((1, 2, 3, 8)), r.choice((1, 2, 4, 7, 8, 16))
    D, qt = r.choice((64, 128)), r.choice((BF16, F16))
    kt, bs = r.choice((qt, qt, FP8)), r.choice((16, 32, 48, 64))
    q_len = r.choice([n for n in (1, 1, 1, 2, 3, 5, 8) if n * G <= 64])
    groups, lens, at = [], [], r.choice((0, 0, 1, 2))
    lens += [r.randrange(0, 300) for _ in range(at)]
    for _ in range(r.randrange(1, 5)):
        n, pages = r.choice((1, 2, 3, 5, 12, 40)), r.choice((0, 1, 2, 5, 17, 40)) * 16 // bs
        groups.append((at, n, pages))
        at += n
        for _ in range(n):
            kind = r.random()
            lens.append(0 if kind < 0.08 else
                        r.randrange(1, pages * bs + 2) if kind < 0.16 else
                        pages * bs + r.choice((0, 1, q_len, 15, 16, 31, 128, 200, 256, 511)))
    lens += [r.randrange(0, 300) for _ in range(r.choice((0, 0, 1, 3)))]
    x = Batch(KVH * G, KVH, D, qt, kt, groups, lens, q_len, bs, extra=r.choice((0, 3)), seed=seed)
    note(f"seed {seed}: H{KVH * G}/KVH{KVH}/D{D} {qt} over {kt}, pages of {bs}, q_len {q_len}, {groups}")
    x.check(x.call(), rows=sorted(r.sample(range(len(lens)), min(12, len(lens)))))


# Calls that the kernel does not take run paged_attention: bit for bit its result.
@pytest.mark.parametrize("name,H,KVH,D,qt,kt,bs,q_len", [
    ("fp32 query", 8, 2, 64, F32, F32, 16, 1), ("fp32 cache", 8, 2, 64, BF16, F32, 16, 1),
    ("fp16 over bf16", 8, 2, 64, F16, BF16, 16, 1), ("head_dim 80", 8, 2, 80, BF16, BF16, 16, 2),
    ("pages of 24", 8, 2, 64, BF16, BF16, 24, 1), ("long chunk", 8, 1, 64, BF16, BF16, 16, 40),
])
def test_other_types_and_layouts(device, name, H, KVH, D, qt, kt, bs, q_len):
    x = Batch(H, KVH, D, qt, kt, [(0, 3, 4)], [150, 120, 110], q_len, bs)
    note(name)
    assert torch.equal(x.call(), x.call(paged_attention))


def test_more_rows_than_the_plan_holds(device):
    x = Batch(2, 1, 64, BF16, BF16, [(0, 1030, 3)], [49 + i % 60 for i in range(1030)], 1)
    note("1030 rows")
    assert torch.equal(x.call(), x.call(paged_attention))
    y = Batch(2, 1, 64, BF16, BF16, [(i, 1, 1) for i in range(0, 1024)], [20] * 1024, 1)
    note("1024 rows and groups")
    y.check(y.call(), rows=[0, 1, 500, 1023])
    z = Batch(2, 1, 64, BF16, BF16, [(0, 1024, 3)], [49 + i % 60 for i in range(1024)], 1)
    z.check(z.call(), rows=[0, 1, 500, 1023])


def test_device_groups_out_of_range(device):
    """Group arrays on the device are not read by the host: values past the bounds count as them."""
    x = Batch(8, 2, 64, BF16, BF16, [(0, 3, 6), (3, 3, 9)], [120, 100, 97, 200, 150, 145], 1)
    want = x.call()
    x.rows = torch.tensor([-5, 3, 2 ** 31 - 1], device=device)
    note("group rows out of range")
    x.pages = torch.tensor([6, 9], device=device)
    assert torch.equal(want, x.call())
    # every page of the table shared: the rows' own parts are empty
    for b in range(3):
        x.table[b] = x.table[0]
        x.table[3 + b] = x.table[3]
    x.lens = [120, 100, 97, 200, 150, 145]
    x.pages = torch.tensor([2 ** 31 - 1, 10 ** 6], device=device)
    x.check(x.call())
    x.pages = torch.tensor([-3, -2 ** 31], device=device)
    x.check(x.call())


@pytest.mark.parametrize("rows", [[0, 4, 2, 6], [3, 1, 0, 0], [6, 6, 6, 2], [2 ** 31 - 1, 0, -7, 4]])
def test_device_groups_out_of_order(device, rows):
    """Group rows on the device that do not ascend: every row by itself."""
    x = Batch(8, 2, 64, BF16, BF16, [], [120, 100, 0, 200, 150, 145], 2)
    x.rows, x.pages = torch.tensor(rows, device=device), torch.tensor([3, 4, 5], device=device)
    note(f"group rows {rows}")
    x.check(x.call())


def test_offsets_past_32_bits(device):
    """Pages whose elements lie past 2^31 in an fp8 pool."""
    x = Batch(8, 8, 128, BF16, FP8, [(0, 2, 3), (2, 2, 5)], [100, 64, 300, 90], 1)
    n = x.kc.shape[0]
    first = 2 ** 31 // (16 * 8 * 128) - n // 2
    pools = []
    for t in (x.kc, x.vc):
        pool = torch.zeros(first + n, 16, 8, 128, dtype=torch.uint8, device=device)
        pool[first:] = t.view(torch.uint8).to(device)
        pools.append(pool.view(FP8))
    note("offsets past 32 bits")
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device)
    out = paged_attention_shared(x.q.to(device), *pools, (x.table + first).to(device), lens, x.rows,
                                 x.pages)
    x.check(out)


def test_refusals(device):
    x = Batch(8, 2, 64, BF16, BF16, [(0, 3, 4)], [150, 120, 110], 1)
    a = [t.to(device) for t in (x.q, x.kc, x.vc, x.table)]
    lens = x.lens
    for rows, pages in (([0, 3], [4, 1]), ([0, 4], [1]), ([2, 1], [1]), ([-1, 2], [1]),
                        ([0, 3], [11]), ([0, 3], [-1]), ([0], [1]), ([0, 1, 2], [1])):
        with pytest.raises(ValueError):
            paged_attention_shared(*a, lens, rows, pages)
    ok = ([0, 3], [4])
    for bad in (dict(out=torch.empty_like(a[0]).float()), dict(out=a[0][:2]),
                dict(out=torch.empty(3, 1, 64, 8, dtype=BF16, device=device).transpose(2, 3))):
        with pytest.raises(ValueError):
            paged_attention_shared(*a, lens, *ok, **bad)
    with pytest.raises(ValueError):
        paged_attention_shared(a[0], a[1], a[2][:3], a[3], lens, *ok)
    with pytest.raises(ValueError):
        paged_attention_shared(*a[:3], a[3][:2], lens, *ok)
    with pytest.raises(ValueError):
        paged_attention_shared(*a, lens[:2], *ok)
    with pytest.raises(ValueError):
        paged_attention_shared(*a, [9999, 1, 1], *ok)
    with pytest.raises(ValueError, match="whole numbers"):
        paged_attention_shared(*a, lens, torch.tensor([0.0, 3.0], device=device), [4])
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_attention_shared(x.q, *a[1:], lens, *ok)
    # an output that is the query: as if it were another
    want = x.call()
    assert torch.equal(want, paged_attention_shared(*a, lens, *ok, out=a[0]))


def test_forward_takes_groups(device):
    x = Batch(8, 2, 64, BF16, BF16, [(0, 3, 6)], [120, 100, 97], 1)
    pa = PagedAttention(8, 2, 64, num_blocks=x.kc.shape[0], block_size=16, dtype=BF16,
                        device=device, kv_dtype=BF16)
    a = [t.to(device) for t in (x.q, x.kc, x.vc, x.table)]
    note("forward")
    for backend in ("sdpa", "triton_flash"):
        got = pa.forward(*a, x.lens, prefix_groups=(x.rows, x.pages), backend=backend)
        assert torch.equal(got, x.call(lens=x.lens))
    plain = paged_attention(*a, x.lens, window=50)
    assert torch.equal(pa.forward(*a, x.lens, window=50, prefix_groups=(x.rows, x.pages)), plain)


def test_streams_and_graphs(device):
    """On a side stream; two graphs on one workspace, replayed in turn over new lengths, groups and
    values, with eager calls of this and other entry points on the same workspace between."""
    x = Batch(14, 2, 64, BF16, BF16, [(0, 4, 20), (4, 4, 6)],
              [500, 400, 330, 321, 200, 150, 100, 97], 1)
    y = Batch(14, 2, 64, BF16, BF16, [(0, 4, 20), (4, 4, 6)],
              [350, 322, 330, 600, 600, 98, 100, 111], 1, seed=3)
    cap = max(x.table.shape[1], y.table.shape[1])
    nb = max(x.kc.shape[0], y.kc.shape[0])
    st = {"q": torch.zeros(8, 1, 14, 64, dtype=BF16, device=device),
          "kc": torch.zeros(nb, 16, 2, 64, dtype=BF16, device=device),
          "vc": torch.zeros(nb, 16, 2, 64, dtype=BF16, device=device),
          "table": torch.full((8, cap), -1, dtype=torch.int32, device=device),
          "lens": torch.zeros(8, dtype=torch.int32, device=device),
          "rows": torch.zeros(3, dtype=torch.int32, device=device),
          "pages": torch.zeros(2, dtype=torch.int32, device=device)}
    ws = torch.zeros(nat.lib().msattn_shared_workspace_bytes(8, 1, 14, 2, 64, cap * 16, 2),
                     dtype=torch.uint8, device=device)
    outs = [torch.empty_like(st["q"]) for _ in range(2)]

    def call(out):
        return paged_attention_shared(st["q"], st["kc"], st["vc"], st["table"], st["lens"],
                                      st["rows"], st["pages"], workspace=ws, out=out)

    def load(z):
        st["q"].copy_(z.q)
        st["kc"][:z.kc.shape[0]].copy_(z.kc)
        st["vc"][:z.vc.shape[0]].copy_(z.vc)
        st["table"].fill_(-1)
        st["table"][:, :z.table.shape[1]].copy_(z.table)
        st["lens"].copy_(torch.tensor(z.lens))
        st["rows"].copy_(torch.tensor(z.rows))
        st["pages"].copy_(torch.tensor(z.pages))

    load(x)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        call(outs[0])
    torch.cuda.current_stream(device).wait_stream(side)
    x.check(outs[0])
    graphs = []
    for out in outs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(out)
        graphs.append(gr)
    for step in range(3):
        for z, gr, out in ((x, graphs[0], outs[0]), (y, graphs[1], outs[1]),
                           (y, graphs[0], outs[0])):
            load(z)
            note(f"replay {step}")
            gr.replay()
            z.check(out)
            assert torch.equal(out, call(None))
            paged_attention(st["q"], st["kc"], st["vc"], st["table"], st["lens"], workspace=ws)
