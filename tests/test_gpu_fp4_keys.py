"""Attention over the 4-bit cache weighs every key once, and with all the digits it says it does
(the contexts and the bound: test_fp4_marks.py, where lost keys and rounder weights are shown to pass
it)."""
import pytest
import torch

from miniserve_amd import paged_attention_fp4
from test_fp4_marks import BF16, F16, F32, SCALE, Marked

pytestmark = pytest.mark.gpu


def call(x, device, lens=None, **kw):
    lens = torch.tensor(x.lens, dtype=torch.int32, device=device) if lens is None else lens
    return paged_attention_fp4(x.q.to(device), *(c.to(device) for c in x.caches),
                               x.table.to(device), lens, scale=SCALE, **kw)


# H, KVH, D, lens, q_len, window
WEIGHTS = {
    "a tile": (8, 2, 64, [16, 40, 1, 0], 1, None),
    "ragged": (14, 2, 128, [300, 33, 700, 64], 1, None),
    "drafts": (16, 2, 64, [300, 95], 4, None),
    "a chunk": (8, 1, 128, [300, 170], 40, None),
    "a window": (8, 2, 96, [500, 333], 3, 70),
    "long": (4, 2, 64, [9000, 20000], 1, None),
}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("name", list(WEIGHTS))
def test_weights_keep_their_digits(device, name, dtype):
    H, KVH, D, lens, q_len, window = WEIGHTS[name]
    x = Marked(H, KVH, D, dtype, lens, q_len)
    print(f"[case] weights {name} {dtype}", flush=True)
    x.check(call(x, device, window=window), window=window)
