"""Contexts over the 4-bit cache whose answers show every key's weight, and what an answer may be off.

Marks. The values of the keys 32 t .. 32 t + 31 hold MARK at dim t mod D, unit normals elsewhere (as
the cache stores them), so that a lost, doubled or misplaced group of keys moves an output at any
length. Queries have one dim that is not zero, so that a score is one exact product.

Bound, for each element. With p the weights in 64 bits, out = sum p_j v_j:
  * a weight is off by a factor within 1 +- C, in numerator and sum alike: C = e^(2 ds) - 1 + 2^-18,
    ds = 8 2^-24 max |s| for the scale's rounding, the multiplication's and the subtraction's (whose
    operands are at most twice the largest score), 2^-18 the hardware's 2^x and the joins': at most
    C / (1 - C) sum p_j |v_j - out|;
  * the numerator alone takes it as parts of bf16, each rounded to nearest (u = 2^-8): it loses
    A = u^2 for the two parts of bf16 and fp16 queries, u^3 for the three of fp32: A sum p_j |v_j|;
  * sums are taken in fp32, 32 keys an instruction, and joined: S = (n / 32 + 40) 2^-23, over
    S (sum p_j |v_j| + |out|);
  * the output is rounded once: eps / 2 |out|, and half of fp16's least step.
"""
import math

import numpy as np
import pytest
import torch

from oracle import dense, fp4

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MARK, GROUP, SCALE = 48.0, 32, 0.25


class Marked:
    """Rows of `lens` keys over a 4-bit cache; what no row may see reads as NaN."""

    def __init__(self, H, KVH, D, dtype, lens, q_len=1, bs=16, extra=0, seed=0):
        g = torch.Generator().manual_seed(seed + 13 * H + D + len(lens))
        B, self.bs, self.lens, self.G = len(lens), bs, list(lens), H // KVH
        need = sum(-(-max(n, 0) // bs) for n in lens) + 3
        perm = torch.randperm(need, generator=g).tolist()
        width = max(1, max(-(-n // bs) for n in lens)) + extra
        self.table = torch.full((B, width), -1, dtype=torch.int32)
        first = torch.zeros(need, dtype=torch.int64)  # position of a page's first token
        seen = np.zeros((need, bs), dtype=bool)
        for b, n in enumerate(lens):
            for c in range(-(-max(n, 0) // bs)):
                page = perm.pop()
                self.table[b, c], first[page] = page, c * bs
                seen[page, :n - c * bs] = True
        k, v = (torch.randn(need, bs, KVH, D, generator=g) for _ in range(2))
        mark = (first[:, None] + torch.arange(bs)) // GROUP % D
        v.scatter_(3, mark[:, :, None, None].expand(need, bs, KVH, 1), MARK)
        self.caches = []
        kept = []
        for x, is_values in ((k, False), (v, True)):
            codes, scale = quantise(x)
            kept.append(fp4.values(codes, scale))
            codes[~seen], scale[~seen] = 15, 255
            self.caches.append(pack(codes, scale, is_values))
        self.k, self.v = kept
        self.q = torch.zeros(B, q_len, H, D)
        dim = torch.randint(0, D, (B, q_len, H, 1), generator=g)
        self.q.scatter_(3, dim, torch.rand(B, q_len, H, 1, generator=g) + 0.5)
        self.q = self.q.to(dtype)

    def keys(self, b):
        """Row b's values of keys and values in 64 bits, and which of them have a page."""
        pages = self.table[b].numpy().copy()
        hole = (pages < 0) | (pages >= self.k.shape[0])
        pages[hole] = 0
        at = np.arange(self.lens[b])
        return (*(x[pages[at // self.bs], at % self.bs] for x in (self.k, self.v)),
                ~hole[at // self.bs])

    def row(self, b, i, h, causal=True, window=None, drop=None):
        """(out, limit) [D] of query (b, i, h); `drop`: keys that the answer is without."""
        k, v, live = self.keys(b)
        keep = dense.keep_mask(self.lens[b], self.q.shape[1], causal, window)[i] & live
        k, v = k[:, h // self.G], v[:, h // self.G]
        s = SCALE * (k @ self.q[b, i, h].double().numpy())
        weigh = keep if drop is None else keep & ~drop
        if not weigh.any():
            return np.zeros(v.shape[1]), np.zeros(v.shape[1])
        p = np.where(weigh, np.exp(np.where(weigh, s - s[weigh].max(), 0.0)), 0.0)
        p /= p.sum()
        v = np.where(keep[:, None], v, 0.0)
        out = p @ v
        if drop is not None:
            return out, None
        dtype = self.q.dtype
        ds = 8 * 2.0 ** -24 * np.abs(s[keep]).max()
        c = math.expm1(2 * ds) + 2.0 ** -18
        a = 2.0 ** (-24 if dtype == F32 else -16)
        sums = (self.lens[b] / 32 + 40) * 2.0 ** -23
        mass = p @ np.abs(v)
        far = p[keep] @ np.abs(v[keep] - out)
        half = torch.finfo(dtype).eps / 2
        least = 2.0 ** -25 if dtype == F16 else 0.0
        return out, 1.01 * (c / (1 - c) * far + a * mass + sums * (mass + np.abs(out))) \
            + half * np.abs(out) + least

    def check(self, got, causal=True, window=None, rows=None):
        got = got.cpu().double().numpy()
        B, T, H, _ = got.shape
        for b in range(B) if rows is None else rows:
            for i in range(T):
                for h in range(H):
                    if self.lens[b] <= 0:
                        assert not got[b, i, h].any()
                        continue
                    out, limit = self.row(b, i, h, causal, window)
                    over = np.abs(got[b, i, h] - out) - limit
                    assert not np.isnan(got[b, i, h]).any() and over.max() <= 0, \
                        (b, i, h, int(over.argmax()), over.max(), limit[over.argmax()])


def quantise(x):
    """fp4.quantise by the exponents of the largest magnitudes: the tests' contexts are long."""
    blocks = x.double().unflatten(-1, (-1, 32))
    top = blocks.abs().amax(-1, keepdim=True)
    mant, exp = torch.frexp(top)  # top = mant 2^exp, mant in [0.5, 1)
    exp = torch.where(top > 0, exp - 3 + (mant > 0.875), -126).clamp(-126, 125)
    y = torch.ldexp(blocks.abs(), -exp)
    code = sum((y > m if i % 2 == 0 else y >= m).to(torch.uint8) for i, m in
               enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)))
    code |= torch.signbit(blocks).to(torch.uint8) << 3
    return code.flatten(-2).numpy(), (exp[..., 0] + 127).to(torch.uint8).numpy()


def pack(codes, scale, is_values):
    """fp4.pack without a loop over elements: the tests' contexts are long."""
    nb, bs, H, D = codes.shape
    pair = torch.from_numpy(codes[..., 0::2] | (codes[..., 1::2] << 4))
    pair = pair.view(nb, bs // 16, 16, H, D // 2).permute(0, 3, 1, 2, 4)  # [nb, H, tiles, 16, D / 2]
    if is_values:
        pair = pair.unflatten(-1, (D // 8, 4)).transpose(3, 4)
    by = torch.from_numpy(scale).view(nb, bs // 16, 16, H, D // 32).permute(0, 3, 1, 4, 2)
    return torch.cat((pair.flatten(3), by.flatten(3)), dim=3).contiguous()


def test_packing():
    x = torch.randn(2, 32, 3, 96, generator=torch.Generator().manual_seed(0))
    x[0, 0, 0, :12] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.0, -5, 5.01, -0.25])
    x[0, 1, 0, :32], x[0, 2, 0, 0], x[0, 3, 0, 0] = 0.0, 7.0, 1e-40
    codes, scale = fp4.quantise(x)
    assert (quantise(x)[0] == codes).all() and (quantise(x)[1] == scale).all()
    for is_values in (False, True):
        assert torch.equal(pack(codes, scale, is_values), fp4.pack(codes, scale, is_values))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [100, 1000, 20000])
def test_lost_keys_are_noticed(dtype, n):
    """Zeros, a missing eighth of the keys, every eighth group missing, one group missing."""
    x = Marked(4, 2, 64, dtype, [n], seed=n)
    key = np.arange(n)
    for h in range(4):
        out, limit = x.row(0, 0, h)
        wrong = [np.zeros_like(out)]
        for drop in (key < n // 8, (key >= n // 2) & (key < n // 2 + n // 8),
                     key // GROUP % 8 == 1, key // GROUP == 1, key // GROUP == (n - 1) // GROUP):
            wrong.append(x.row(0, 0, h, drop=drop)[0])
        for i, w in enumerate(wrong):
            assert (np.abs(w - out) > limit).any(), (h, i)
        rounded = torch.from_numpy(out).to(dtype).double().numpy()
        assert (np.abs(rounded - out) <= limit).all()


def test_weights_of_eight_bits_are_noticed():
    """What a bf16 query's weights lose if each is rounded to bf16 once, numerator and sum alike."""
    for n in (40, 300, 1000):
        x = Marked(8, 2, 64, BF16, [n], seed=n)
        k, v, _ = x.keys(0)
        over = 0
        for h in range(8):
            s = SCALE * (k[:, h // 4] @ x.q[0, 0, h].double().numpy())
            p = torch.from_numpy(np.exp(s - s.max())).to(BF16).double().numpy()
            out, limit = x.row(0, 0, h)
            got = torch.from_numpy(p @ v[:, h // 4] / p.sum()).to(BF16).double().numpy()
            over += int((np.abs(got - out) > 1.5 * limit).sum())
        assert over > 5, (n, over)
