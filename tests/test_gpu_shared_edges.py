"""Attention behind shared prefixes at the ends of its arguments."""
import pytest
import torch

from miniserve_amd import paged_attention_shared, shared
from test_gpu_shared import BF16, Batch, note

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
