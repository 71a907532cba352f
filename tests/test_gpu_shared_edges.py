"""Attention behind shared prefixes at the ends of its arguments."""
import pytest
import torch

from miniserve_amd import paged_attention_shared, shared
from test_gpu_shared import BF16, F16, FP8, Batch, note

pytestmark = pytest.mark.gpu


def test_device_groups_past_32_bits(device):
    """int64 group rows and pages past int32 count as the nearest bound, not modulo 2^32."""
    x = Batch(8, 2, 64, BF16, BF16, [(0, 3, 6), (3, 3, 9)], [120, 100, 97, 200, 150, 145], 1)
    want = x.call()
    note("group rows past 32 bits")
    x.rows = torch.tensor([-2 ** 40, 3, 2 ** 31], device=device)
    x.pages = torch.tensor([6, 9], device=device)
    assert torch.equal(want, x.call())
    # all pages shared: 2^32 + 1 pages are the table's, not one; -2^32 + 4 none, not four
    for b in range(3):
        x.table[b], x.table[3 + b] = x.table[0], x.table[3]
    x.rows = [0, 3, 6]
    note("prefix pages past 32 bits")
    got = {}
    for name, pages in (("wide", [2 ** 32 + 1, -2 ** 32 + 4]), ("bounds", [x.table.shape[1], 0])):
        x.pages = torch.tensor(pages, device=device)
        got[name] = x.call()
        x.check(got[name])
    assert torch.equal(got["wide"], got["bounds"])


def test_no_group_on_another_device_than_the_current_one(device, monkeypatch):
    """A call without a group runs paged_attention with the tensors' device current."""
    x = Batch(8, 2, 64, BF16, BF16, [(0, 3, 6)], [120, 100, 97], 1)
    x.rows, x.pages = [], []
    inside, seen = [], []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            inside.append(self.dev)

        def __exit__(self, *e):
            inside.pop()

    real = shared.paged_attention
    monkeypatch.setattr(shared, "paged_attention", lambda *a, **kw: (seen.append(list(inside)), real(*a, **kw))[1])
    args = [t.to(device) for t in (x.q, x.kc, x.vc, x.table)]
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 7)
    monkeypatch.setattr(torch.cuda, "device", Device)
    note("another device")
    paged_attention_shared(*args, lens, [], [])
    assert seen == [[device]] and not inside


def test_refuses_a_workspace_elsewhere(device):
    x = Batch(8, 2, 64, BF16, BF16, [(0, 3, 6)], [120, 100, 97], 1)
    note("workspace elsewhere")
    for ws in (torch.zeros(64 << 20, dtype=torch.uint8),
               torch.zeros(128 << 20, dtype=torch.uint8, device=device)[::2]):
        with pytest.raises(ValueError, match="workspace must"):
            x.call(workspace=ws)


@pytest.mark.parametrize("H,KVH,D,qt,kt,T", [
    (4, 2, 64, BF16, BF16, 3), (28, 4, 128, F16, F16, 8), (16, 1, 64, F16, FP8, 4),
    (32, 8, 128, BF16, BF16, 5), (8, 2, 128, BF16, FP8, 7), (16, 4, 128, BF16, BF16, 16),
    (14, 2, 64, F16, F16, 2),
])
def test_values_that_only_later_drafts_see(device, H, KVH, D, qt, kt, T):
    """NaN in the last key's values and an infinite value in the key before it: the drafts that see
    them have NaN and infinity at those dims of those heads, everything else is bit for bit what it
    is without them. The rows' drafts straddle blocks of 32 keys and tiles."""
    x = Batch(H, KVH, D, qt, kt, [(0, 3, 4), (3, 2, 2)], [97, 130, 194, 80, 289], T)
    clean = x.call().cpu()
    x.check(clean)
    bad = [(1, 3, float("nan"))] + ([] if kt == FP8 else [(2, 5, float("inf")), (2, 6, float("-inf"))])
    head = KVH - 1
    want = clean.clone().view(x.B, T, KVH, H // KVH, D)
    for b, n in enumerate(x.lens):
        for back, dim, value in bad:
            page, slot = int(x.table[b, (n - back) // 16]), (n - back) % 16
            x.vc.view(torch.uint8 if kt == FP8 else kt)[page, slot, head, dim] = \
                0x7f if kt == FP8 else value
            want[b, T - back:, head, :, dim] = value
    note(f"values of later drafts, {T} tokens, {kt}")
    got = x.call().cpu().view_as(want)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
