"""That attention behind shared prefixes (paged_attention_shared) weighs every key once, at any
length: values carry marks that a lost, doubled or misplaced block of 32 keys moves by more than
the kernel may err, and every reference is shown to notice that before the kernel is compared.

Marks. The values of the keys 32 t .. 32 t + 31 hold MARK at dim t mod D, unit normals elsewhere.

Bound, for each element. With p the weights in 64 bits and out = sum p_j v_j: the kernel's weights
are off by a factor within 1 +- E, E = u + (e^(2 ds) - 1) + 2^-18, of which u = eps / 2 rounds them
to the query type, ds = (D + 8) 2^-24 |scale| |q||k| bounds a score's error (products, D additions,
the scale) and 2^-18 the hardware's 2^x and the rounding of its argument. They are divided by the sum
of the same rounded weights, so that the error is at most E / (1 - E) sum p_j |v_j - out|. fp16
weights below 2^-14 are rounded by 2^-25 beside a largest one of 1 or more: 2^-25 sum |v_j - out| / L
more, L the sum of the weights over their largest. The sums are taken in fp32, 32 keys an
instruction, rescaled at most once each, over at most 512 pieces: (n / 16 + 1100) 2^-24 (sum p_j
|v_j| + |out|). The output is rounded once: u |out|, and half of fp16's least step.
"""
import pytest
import torch

from miniserve_amd import _native as nat, paged_attention, paged_attention_shared

pytestmark = pytest.mark.gpu
F32, F16, BF16, FP8 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
MARK, BLOCK, BS = 56.0, 32, 16


def note(msg: str) -> None:
    print(f"[case] {msg}", flush=True)


class Marked:
    """Rows in groups [(first row, rows, prefix pages)] over a pool that holds no page more than
    they need, in shuffled order; `own` keys a row past its group's prefix."""

    def __init__(self, H, KVH, D, qt, kt, groups, own, q_len=1, seed=0):
        g = torch.Generator().manual_seed(seed + 13 * H + D + len(own))
        B = len(own)
        self.rows, self.pages, first = [groups[0][0]], [], [0] * B
        for r0, n, p in groups:
            assert r0 == self.rows[-1]
            self.rows.append(r0 + n)
            self.pages.append(p)
            first[r0:r0 + n] = [p] * n
        self.lens = [f * BS + n for f, n in zip(first, own)]
        self.W = max(-(-n // BS) for n in self.lens)
        need = sum(self.pages) + sum(-(-n // BS) for n in own)
        ids = torch.randperm(need, generator=g).to(torch.int32)
        self.table = torch.full((B, self.W), -1, dtype=torch.int32)
        place = torch.zeros(need, dtype=torch.int64)  # the page's place in its sequence
        at = 0
        for r0, n, p in groups:
            self.table[r0:r0 + n, :p] = ids[at:at + p]
            place[ids[at:at + p].long()] = torch.arange(p)
            at += p
        for b, n in enumerate(own):
            w = -(-n // BS)
            self.table[b, first[b]:first[b] + w] = ids[at:at + w]
            place[ids[at:at + w].long()] = torch.arange(first[b], first[b] + w)
            at += w
        k, v = (torch.randn(need, BS, KVH, D, generator=g) for _ in range(2))
        block = (place[:, None] * BS + torch.arange(BS)) // BLOCK % D
        v.scatter_(3, block[:, :, None, None].expand(need, BS, KVH, 1), MARK)
        self.kc, self.vc = k.to(kt), v.to(kt)
        self.q = torch.randn(B, q_len, H, D, generator=g).to(qt)

    def call(self, device, fn=paged_attention_shared, **kw):
        args = [t.to(device) for t in (self.q, self.kc, self.vc, self.table)]
        lens = torch.tensor(self.lens, dtype=torch.int32, device=device)
        if fn is paged_attention:
            return fn(*args, lens, **kw)
        return fn(*args, lens, self.rows, self.pages, **kw)

    def reference(self, b, notices=True):
        """(output, bound) of row b [q_len, H, D] in 64 bits; `notices`: that every block of keys,
        dropped or doubled, moves some element by more than twice its bound is checked."""
        q = self.q[b].double()
        T, H, D = q.shape
        KVH, n = self.kc.shape[2], self.lens[b]
        at = self.table[b, :-(-n // BS)].long()
        k, v = (c[at].reshape(-1, KVH, D)[:n].to(self.q.dtype).double() for c in (self.kc, self.vc))
        scale, u = D ** -0.5, torch.finfo(self.q.dtype).eps / 2
        out, bound = torch.zeros(T, H, D).double(), torch.zeros(T, H, D).double()
        for kvh in range(KVH):
            heads = slice(kvh * (H // KVH), (kvh + 1) * (H // KVH))
            x = (q[:, heads].reshape(-1, D) @ k[:, kvh].T) * scale
            last = torch.arange(n - T, n).repeat_interleave(H // KVH)
            x = x.masked_fill(torch.arange(n) > last[:, None], -torch.inf)
            w = torch.exp(x - x.amax(1, keepdim=True))
            L = w.sum(1, keepdim=True)
            p = w / L
            vk = v[:, kvh]
            o = p @ vk
            away = torch.stack([p[r] @ (vk - o[r]).abs() for r in range(len(p))])
            ds = (D + 8) * 2.0 ** -24 * scale * q[:, heads].reshape(-1, D).norm(dim=1) * \
                k[:, kvh].norm(dim=1).max()
            E = (u + torch.expm1(2 * ds) + 2.0 ** -18)[:, None]
            e = E / (1 - E) * away + u * o.abs() * (1 + u) + \
                (n / 16 + 1100) * 2.0 ** -24 * (p @ vk.abs() + o.abs())
            if self.q.dtype == F16:
                seen = (p > 0).double()
                far = torch.stack([seen[r] @ (vk - o[r]).abs() for r in range(len(p))])
                e = e + 2.0 ** -25 * far / L + 2.0 ** -25
            if notices:
                blocks = -(-n // BLOCK)
                pad = blocks * BLOCK - n
                pb = torch.nn.functional.pad(p, (0, pad)).view(-1, blocks, BLOCK)
                vb = torch.nn.functional.pad(vk, (0, 0, 0, pad)).view(blocks, BLOCK, D)
                S = torch.einsum("rtj,tjd->rtd", pb, vb)
                P = pb.sum(2, keepdim=True)
                move = (P * o[:, None] - S).abs()
                whole = P[..., 0] > 0
                for what, gone in (("dropped", move / (1 - P).clamp(min=1e-12)),
                                   ("doubled", move / (1 + P))):
                    seen = (gone > 2 * e[:, None]).any(2) | ~whole
                    # (a last block of a few keys weighs too little: the others count)
                    few = torch.arange(blocks) * BLOCK + BLOCK > n - T
                    assert bool((seen | few).all()), f"row {b}: a block {what} would not show"
            out[:, heads] = o.view(T, -1, D)
            bound[:, heads] = e.view(T, -1, D)
        return out, bound

    def check(self, out, rows=None, notices=True):
        out = out.cpu().double()
        for b in range(len(self.lens)) if rows is None else rows:
            want, bound = self.reference(b, notices)
            over = ((out[b] - want).abs() - bound).max().item()
            assert over <= 0, f"row {b} of {self.lens[b]} keys: {over:.3e} over the bound"


# name -> (H, KVH, D, query, cache, groups, own keys, q_len)
CASES = {
    "one KV head": (4, 1, 128, BF16, BF16, [(0, 3, 600)], [100, 1400, 10400], 1),
    "one KV head, 64 dims": (2, 1, 64, F16, F16, [(0, 2, 1100)], [100, 12401], 1),
    "fp8": (4, 1, 128, F16, FP8, [(0, 2, 600)], [100, 9401], 1),
    "fp8, 64 dims": (4, 2, 64, BF16, FP8, [(0, 2, 300), (2, 3, 500)], [64, 4001, 200, 31, 900], 1),
    "groups and a loose row": (8, 4, 128, BF16, BF16, [(1, 2, 70), (3, 4, 250)],
                               [3333, 100, 2000, 700, 90, 1500, 33], 1),
    "drafts": (14, 2, 128, F16, F16, [(0, 6, 160)], [100, 230, 400, 90, 1000, 64], 4),
    "129 query rows": (43, 1, 128, BF16, BF16, [(0, 3, 300)], [100, 700, 64], 1),
    "fp8, 200 query rows": (40, 1, 128, BF16, FP8, [(0, 5, 200)], [64, 100, 600, 128, 1000], 1),
    "64 query rows": (16, 1, 64, F16, F16, [(0, 2, 400)], [400, 2000], 4),
}


@pytest.mark.parametrize("name", list(CASES))
def test_every_key_once(device, name):
    x = Marked(*CASES[name])
    note(f"every key once, {name}")
    x.check(x.call(device))


def test_shares_of_more_than_one_window_wide_units(device):
    """A group of 1024 rows of 8 query rows a KV head behind 8192 keys: 64 blocks of 128 query rows,
    8 KV heads and 64 tiles of 128 keys, 128 tiles a share or more where workgroups plan 64 tiles at
    a time."""
    x = Marked(64, 8, 128, BF16, BF16, [(0, 1024, 512)], [16 + b % 17 for b in range(1024)])
    note("wide units past a window")
    x.check(x.call(device), rows=[0, 511, 1023])


def test_shares_of_more_than_one_window_narrow_units(device):
    """1024 rows of 32 KV heads, one query row each, most of one tile: 128 units a share or more, and
    each is joined by the waves that split its keys, at the last tile of a window too."""
    own = [300 + 77 * (b % 9) if b % 16 == 5 else 16 + b % 25 for b in range(1024)]
    x = Marked(32, 32, 64, BF16, BF16, [(0, 2, 40), (2, 3, 0)], own)
    note("narrow units past a window")
    # (rows of so few keys: a block is nearly all that there is, and shows)
    x.check(x.call(device), rows=[0, 1, 5, 21, 500, 501, 1013, 1023], notices=False)


@pytest.mark.parametrize("H,q_len,taken", [(16, 4, True), (64, 1, True), (65, 1, False), (13, 5, False)])
def test_query_rows_at_the_dispatch(device, H, q_len, taken):
    """Up to 64 query rows a KV head and batch row the kernel plans its work behind the workspace's
    header; past them the call is paged_attention's, bit for bit."""
    x = Marked(H, 1, 64, BF16, BF16, [(0, 3, 30)], [40, 200, 77], q_len)
    cap = x.W * BS
    plan = (64 + 4096) * 4
    ws = torch.zeros(nat.lib().msattn_shared_workspace_bytes(3, q_len, H, 1, 64, cap, 1),
                     dtype=torch.uint8, device=device)
    note(f"{H * q_len} query rows")
    out = x.call(device, workspace=ws)
    if taken:
        assert ws[plan:plan + 4].any()  # the cost of a share, never zero
        x.check(out)
    else:
        assert torch.equal(out, x.call(device, paged_attention))
