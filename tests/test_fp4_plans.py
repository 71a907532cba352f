"""How msattn_paged_attention_fp4 cuts calls: a geometry for every kernel that is compiled, which
test_gpu_fp4_plans.py runs. A change of the cost model that takes a kernel from them shows here."""
import ctypes

import numpy as np
import pytest
import torch

from miniserve_amd import _native as nat

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DEALT, PARTS, LIST = 0, 1, 2

# type, D, (way, blocks of 16 rows, waves a unit, parts), heads, KV heads, rows, longest context,
# tokens of the table, q_len, block size, causal, window
PLANS = [
    (BF16, 32, (0, 1, 1, 1), 34, 2, 1, 137, 192, 642, 48, True, None),
    (BF16, 64, (0, 1, 2, 1), 17, 1, 2, 4167, 4864, 2, 64, True, 3),
    (BF16, 64, (0, 1, 4, 1), 17, 1, 5, 579, 704, 51, 16, True, None),
    (BF16, 32, (0, 1, 8, 1), 3, 1, 2, 7007, 7648, 471, 32, False, None),
    (BF16, 32, (1, 1, 8, 6), 8, 1, 2, 3855, 7936, 1, 256, True, 1338),
    (BF16, 64, (2, 1, 8, 1), 132, 12, 11, 1650, 6272, 1, 64, True, None),
    (BF16, 32, (2, 1, 8, 1), 1, 1, 129, 2588, 7344, 5, 48, True, None),
    (BF16, 64, (0, 2, 1, 1), 60, 3, 1, 217, 272, 668, 16, False, None),
    (BF16, 64, (0, 2, 2, 1), 17, 1, 2, 4359, 6656, 580, 256, True, 762),
    (BF16, 32, (0, 2, 4, 1), 3, 1, 5, 4820, 6560, 680, 32, True, 1727),
    (BF16, 32, (0, 2, 8, 1), 6, 1, 2, 5932, 8960, 509, 32, True, 884),
    (BF16, 64, (1, 2, 8, 30), 1, 1, 2, 4583, 7616, 30, 16, True, None),
    (BF16, 64, (2, 2, 8, 1), 198, 11, 13, 2006, 7936, 1, 16, True, None),
    (BF16, 32, (2, 2, 8, 1), 40, 2, 68, 4911, 7872, 1, 16, True, None),
    (BF16, 32, (2, 2, 8, 1), 13, 1, 1, 6538, 7680, 375, 32, True, None),
    (BF16, 32, (0, 4, 1, 1), 20, 1, 26, 578, 592, 189, 16, True, None),
    (BF16, 64, (0, 4, 2, 1), 18, 1, 18, 662, 1024, 144, 256, True, None),
    (BF16, 64, (0, 4, 4, 1), 17, 1, 5, 4257, 5888, 296, 256, True, None),
    (BF16, 128, (0, 1, 1, 1), 12, 2, 2, 55, 64, 684, 64, True, None),
    (BF16, 96, (0, 1, 2, 1), 4, 1, 2, 3888, 4864, 5, 16, True, 7),
    (BF16, 128, (0, 1, 4, 1), 2, 1, 2, 63, 64, 14, 64, True, None),
    (BF16, 128, (0, 1, 8, 1), 2, 1, 2, 2129, 2272, 11, 16, True, None),
    (BF16, 96, (1, 1, 8, 17), 1, 1, 2, 3209, 4160, 5, 16, False, None),
    (BF16, 128, (2, 1, 8, 1), 10, 10, 13, 1816, 6928, 3, 16, True, None),
    (BF16, 96, (2, 1, 8, 1), 9, 3, 95, 885, 3360, 1, 32, True, None),
    (BF16, 128, (0, 2, 1, 1), 30, 3, 2, 53, 64, 681, 64, True, None),
    (BF16, 128, (0, 2, 2, 1), 20, 1, 6, 485, 928, 188, 16, True, None),
    (BF16, 128, (0, 2, 4, 1), 5, 1, 2, 1955, 3008, 880, 32, True, 696),
    (BF16, 128, (0, 2, 8, 1), 7, 1, 2, 2258, 3600, 341, 48, True, None),
    (BF16, 96, (1, 2, 8, 19), 5, 1, 2, 3061, 4800, 4, 32, True, None),
    (BF16, 128, (2, 2, 8, 1), 154, 11, 12, 2103, 6560, 2, 32, True, None),
    (BF16, 128, (2, 2, 8, 1), 9, 1, 86, 900, 13872, 3, 48, True, None),
    (BF16, 96, (2, 2, 8, 1), 10, 1, 1, 3814, 6992, 449, 16, True, None),
    (BF16, 128, (0, 4, 1, 1), 40, 2, 5, 1176, 1792, 569, 256, True, None),
    (BF16, 128, (0, 4, 2, 1), 15, 1, 18, 628, 800, 172, 32, True, None),
    (BF16, 128, (0, 4, 4, 1), 20, 1, 3, 2747, 3968, 434, 16, True, None),
    (BF16, 256, (0, 1, 1, 1), 18, 3, 2, 57, 64, 470, 64, True, None),
    (BF16, 192, (0, 1, 2, 1), 18, 1, 2, 47, 48, 1, 48, False, None),
    (BF16, 224, (0, 1, 4, 1), 11, 1, 2, 85, 96, 6, 16, True, None),
    (BF16, 224, (0, 1, 8, 1), 14, 1, 2, 1007, 1024, 2, 256, False, None),
    (BF16, 224, (1, 1, 8, 8), 1, 1, 2, 1249, 1792, 2, 256, False, None),
    (BF16, 192, (2, 1, 8, 1), 7, 7, 13, 600, 17728, 8, 64, False, None),
    (BF16, 160, (2, 1, 8, 1), 2, 1, 93, 1200, 17392, 1, 16, True, None),
    (BF16, 192, (2, 1, 8, 1), 22, 2, 1, 5000, 17664, 99, 32, True, None),
    (F16, 32, (0, 1, 1, 1), 21, 3, 2, 149, 208, 394, 16, False, None),
    (F16, 64, (0, 1, 2, 1), 2, 1, 2, 4134, 5088, 35, 16, True, 7),
    (F16, 64, (0, 1, 4, 1), 5, 1, 2, 4621, 7248, 4, 48, True, 54),
    (F16, 64, (0, 1, 8, 1), 15, 1, 2, 2247, 2256, 6, 48, True, None),
    (F16, 64, (1, 1, 8, 8), 6, 1, 2, 4311, 4352, 1, 256, True, 1812),
    (F16, 64, (2, 1, 8, 1), 36, 9, 15, 2158, 7840, 3, 16, True, None),
    (F16, 32, (2, 1, 8, 1), 2, 2, 67, 2232, 8048, 1, 16, False, None),
    (F16, 32, (0, 2, 1, 1), 15, 1, 4, 6009, 7424, 684, 256, True, 74),
    (F16, 32, (0, 2, 2, 1), 15, 1, 5, 2689, 2944, 352, 64, True, None),
    (F16, 64, (0, 2, 4, 1), 9, 1, 2, 4786, 4800, 775, 16, True, None),
    (F16, 64, (0, 2, 8, 1), 20, 1, 2, 4954, 5952, 119, 32, True, None),
    (F16, 64, (1, 2, 8, 30), 5, 1, 2, 4871, 7488, 4, 32, False, None),
    (F16, 64, (2, 2, 8, 1), 7, 7, 20, 2792, 7392, 23, 32, False, None),
    (F16, 32, (2, 2, 8, 1), 2, 2, 71, 3750, 7296, 21, 32, True, None),
    (F16, 64, (2, 2, 8, 1), 7, 1, 1, 3943, 6688, 621, 16, True, None),
    (F16, 128, (0, 1, 1, 1), 30, 5, 1, 61, 64, 549, 64, True, None),
    (F16, 128, (0, 1, 2, 1), 14, 1, 5, 250, 256, 135, 256, True, None),
    (F16, 128, (0, 1, 4, 1), 6, 1, 2, 95, 96, 13, 32, True, None),
    (F16, 96, (0, 1, 8, 1), 1, 1, 2, 1473, 1792, 27, 256, True, None),
    (F16, 128, (1, 1, 8, 12), 2, 1, 2, 2302, 2896, 1, 16, False, None),
    (F16, 96, (2, 1, 8, 1), 140, 10, 13, 2484, 6208, 1, 16, True, None),
    (F16, 96, (2, 1, 8, 1), 4, 1, 130, 2034, 8112, 3, 48, True, None),
    (F16, 128, (2, 1, 8, 1), 2, 1, 1, 6000, 19104, 683, 32, False, None),
    (F16, 96, (0, 2, 1, 1), 171, 9, 1, 209, 224, 208, 16, False, None),
    (F16, 128, (0, 2, 2, 1), 68, 4, 3, 354, 576, 99, 16, True, None),
    (F16, 128, (0, 2, 4, 1), 7, 1, 2, 947, 1648, 812, 16, True, None),
    (F16, 128, (0, 2, 8, 1), 20, 1, 2, 2175, 2224, 132, 16, True, None),
    (F16, 160, (0, 1, 1, 1), 8, 1, 4, 107, 128, 531, 64, False, None),
    (F16, 160, (0, 1, 2, 1), 17, 1, 2, 48, 48, 1, 48, False, None),
    (F16, 224, (0, 1, 4, 1), 9, 1, 2, 64, 64, 2, 64, True, None),
    (F16, 192, (0, 1, 8, 1), 7, 1, 2, 1103, 1152, 3, 16, True, None),
    (F16, 256, (1, 1, 8, 6), 1, 1, 2, 1147, 1472, 2, 64, True, None),
    (F16, 256, (2, 1, 8, 1), 12, 4, 22, 700, 13824, 2, 64, True, None),
    (F16, 192, (2, 1, 8, 1), 4, 2, 75, 500, 17856, 1, 64, True, None),
    (F16, 192, (2, 1, 8, 1), 1, 1, 5, 3000, 19456, 423, 64, False, None),
    (F32, 64, (0, 1, 1, 1), 12, 2, 1, 16, 16, 10, 16, False, None),
    (F32, 32, (0, 1, 2, 1), 35, 5, 1, 491, 512, 357, 64, True, None),
    (F32, 32, (0, 1, 4, 1), 9, 1, 2, 5956, 7936, 2, 32, True, 87),
    (F32, 32, (0, 1, 8, 1), 9, 1, 2, 4929, 8704, 156, 256, True, None),
    (F32, 32, (1, 1, 8, 6), 1, 1, 2, 4918, 8064, 6, 32, True, 1457),
    (F32, 64, (2, 1, 8, 1), 3, 3, 46, 1809, 6912, 3, 256, False, None),
    (F32, 64, (2, 1, 8, 1), 8, 2, 69, 2090, 8304, 1, 48, True, None),
    (F32, 32, (0, 2, 1, 1), 40, 2, 3, 721, 1040, 446, 16, True, None),
    (F32, 32, (0, 2, 2, 1), 14, 1, 3, 3200, 3328, 584, 256, False, None),
    (F32, 64, (0, 2, 4, 1), 15, 1, 2, 1483, 1536, 369, 256, True, None),
    (F32, 32, (0, 2, 8, 1), 13, 1, 2, 6335, 7424, 201, 256, True, None),
    (F32, 64, (1, 2, 8, 34), 5, 1, 2, 4234, 8592, 5, 48, True, None),
    (F32, 64, (2, 2, 8, 1), 15, 5, 26, 2569, 6656, 8, 256, True, None),
    (F32, 64, (2, 2, 8, 1), 14, 2, 72, 1932, 7296, 3, 64, True, None),
    (F32, 64, (2, 2, 8, 1), 14, 1, 3, 3386, 8448, 113, 256, True, None),
    (F32, 128, (0, 1, 1, 1), 5, 1, 3, 16, 16, 12, 16, True, None),
    (F32, 128, (0, 1, 2, 1), 5, 1, 2, 321, 384, 922, 64, False, None),
    (F32, 128, (0, 1, 4, 1), 10, 1, 2, 96, 96, 2, 32, False, None),
    (F32, 96, (0, 1, 8, 1), 2, 1, 2, 3353, 6336, 2, 48, True, 426),
    (F32, 128, (1, 1, 8, 13), 1, 1, 2, 2159, 3312, 3, 48, True, None),
    (F32, 128, (2, 1, 8, 1), 36, 9, 15, 1650, 6592, 3, 64, True, None),
    (F32, 128, (2, 1, 8, 1), 5, 1, 89, 900, 13248, 3, 16, True, None),
    (F32, 96, (2, 1, 8, 1), 2, 1, 2, 4000, 13440, 582, 64, True, None),
    (F32, 160, (0, 1, 1, 1), 11, 1, 2, 16, 16, 6, 16, True, None),
    (F32, 224, (0, 1, 2, 1), 34, 2, 2, 201, 256, 134, 256, True, None),
    (F32, 224, (0, 1, 4, 1), 34, 2, 1, 93, 96, 1, 48, False, None),
    (F32, 192, (0, 1, 8, 1), 18, 1, 2, 1099, 1152, 1, 16, True, None),
    (F32, 160, (1, 1, 8, 18), 1, 1, 2, 1851, 4384, 3, 32, True, None),
    (F32, 192, (2, 1, 8, 1), 16, 8, 11, 500, 13408, 4, 16, True, None),
    (F32, 192, (2, 1, 8, 1), 2, 1, 100, 900, 19536, 3, 48, False, None),
    (F32, 224, (2, 1, 8, 1), 6, 1, 1, 6000, 13888, 356, 64, False, None),
    (BF16, 128, (2, 1, 8, 1), 24, 8, 50, 4500, 12288, 4, 16, True, 3500),
    (F32, 64, (2, 1, 8, 1), 8, 4, 100, 7000, 12288, 2, 16, True, 5800),
    (F16, 64, (2, 1, 8, 1), 24, 8, 50, 7000, 12288, 2, 32, True, 6000),
]


def named(c):
    (way, ct, wk, _), window = c[2], c[11]
    return f"{str(c[0])[6:]}-{c[1]}-{('dealt', 'parts', 'list')[way]}-{ct}-{wk}-{c[3]}x{c[5]}x{c[8]}" + \
        ("" if c[10] else "-all") + (f"-w{window}" if window else "")


def lens_of(c):
    """Contexts of a case: the longest, none, one, fewer than queries, and so on."""
    B, hi, q_len = c[5], c[6], c[8]
    some = [hi, 1, 0, hi // 2, max(1, q_len - 1), hi // 5, hi - 3, 17]
    lens = [some[b] if b < 8 else (hi * (b * 37 % 101) // 101 if b % 8 == 0 else hi // 40 + b)
            for b in range(B)]
    return [max(0, min(hi, n)) for n in lens]


def plan(dtype, D, H, KVH, B, cap, q_len, causal, window):
    p = (ctypes.c_int * 4)()
    status = nat.lib().msattn_fp4_plan(B, q_len, H, KVH, D, cap, int(causal), window or 0,
                                       nat.DTYPE_CODES[dtype], p)
    return tuple(p) if status == nat.OK else status


def plan_of(c):
    dtype, D, _, H, KVH, B, _, cap, q_len, _, causal, window = c
    return plan(dtype, D, H, KVH, B, cap, q_len, causal, window)


@pytest.mark.parametrize("c", PLANS, ids=named)
def test_plan(c):
    assert plan_of(c) == c[2] and c[7] % c[9] == 0 and c[6] <= c[7]


def test_every_kernel_has_a_case():
    """By what fp4_max_ct and fp4_list_ct allow; a list's plan in registers and in LDS, of one row block
    a row and of several."""
    have = {(c[0], 64 if c[1] <= 64 else 128 if c[1] <= 128 else 256, *c[2][:3]) for c in PLANS}
    want = set()
    for dtype, parts in ((BF16, 1), (F16, 2), (F32, 3)):
        for dims in (64, 128, 256):
            most = 1 if dims > 128 or (dims > 64 and parts == 3) else (4 if parts == 1 else 2)
            listed = 1 if dims > 128 or (dims > 64 and parts > 1) else 2
            for ct in (1, 2, 4):
                if ct <= most:
                    want |= {(dtype, dims, DEALT, ct, wk) for wk in (1, 2, 4, 8) if ct * wk < 32}
                if ct <= listed:
                    want |= {(dtype, dims, way, ct, 8) for way in (PARTS, LIST)}
    assert have == want
    lists = [c for c in PLANS if c[2][0] == LIST]
    rows = lambda c: c[8] * c[3] // c[4] / (16 * c[2][1])
    for dtype in (BF16, F16, F32):
        of = [c for c in lists if c[0] == dtype]
        assert any(rows(c) <= 1 and c[5] <= 64 for c in of) and any(rows(c) <= 1 and c[5] > 64 for c in of)
        assert any(rows(c) > 1 for c in of) and any(c[11] for c in of) and any(not c[10] for c in of)


@pytest.mark.parametrize("bad,status", [
    (dict(B=0), 1), (dict(H=3), 1), (dict(D=48), 1), (dict(cap=-1), 1), (dict(window=-1), 1),
    (dict(cap=(1 << 30) + 1), 2), (dict(B=1 << 24), 2)], ids=str)
def test_plan_refuses(bad, status):
    args = {**dict(dtype=BF16, D=64, H=8, KVH=2, B=4, cap=100, q_len=1, causal=True, window=None), **bad}
    assert plan(**args) == status


def test_plan_refuses_no_place_for_it():
    assert nat.lib().msattn_fp4_plan(1, 1, 1, 1, 64, 100, 1, 0, nat.BF16, None) == 1


@pytest.mark.parametrize("n", [700, 20000])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_lost_keys_are_noticed(dtype, n):
    """The check of test_gpu_fp4_plans.py on answers in 64 bits, rounded: passed as they are, not
    without a group of keys, nor without a wave's or an eighth of them, nor as zeros."""
    from test_fp4_marks import GROUP, Marked
    from test_gpu_fp4_plans import check
    x = Marked(4, 2, 64, dtype, [n, 50, 0], 2, seed=3)
    key = np.arange(n)
    answer = np.zeros((3, 2, 4, 64))
    for b, i, h in np.ndindex(2, 2, 4):
        answer[b, i, h] = x.row(b, i, h)[0]
    cpu = torch.device("cpu")
    check(cpu, x, torch.from_numpy(answer).to(dtype), True, None)
    for drop in (key // GROUP == 5, key // GROUP % 8 == 2, (key >= n // 2) & (key < n // 2 + n // 8)):
        wrong = answer.copy()
        wrong[0, 1, 3] = x.row(0, 1, 3, drop=drop)[0]
        with pytest.raises(AssertionError):
            check(cpu, x, torch.from_numpy(wrong).to(dtype), True, None)
    with pytest.raises(AssertionError):
        check(cpu, x, torch.zeros(3, 2, 4, 64, dtype=dtype), True, None)
