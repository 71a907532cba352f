"""Edges of the 4-bit cache's entry points: values, arguments and places that lie apart from a run's."""
import pytest
import torch

from miniserve_amd import allocate_fp4_cache, paged_attention_fp4, write_kv_fp4

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("q_len", [1, 20])
@pytest.mark.parametrize("dtype,bits", [(F32, 0x7F800001), (F32, 0x7F80FFFF), (F32, -0x7FFFFF), (F32, 0x7FC00000),
                                        (F16, 0x7C01), (F16, 0x7E00), (BF16, 0x7F81)])
def test_every_nan_of_a_query_stays_one(device, dtype, bits, q_len):
    """Keys that are negative in the NaN's dim: an infinity there would hide every one of them."""
    KVH, D, n = 2, 64, 70
    kc, vc = allocate_fp4_cache(8, 16, KVH, D, device=device)
    table = torch.arange(5, dtype=torch.int32, device=device).view(1, 5)
    k = torch.full((1, n, KVH, D), -1.0, device=device)
    v = torch.randn(1, n, KVH, D, device=device, generator=torch.Generator(device).manual_seed(1))
    write_kv_fp4(k, v, kc, vc, table)
    q = torch.ones(1, q_len, 4, D, dtype=dtype, device=device)
    ints = q.view(torch.int32 if dtype == F32 else torch.int16)
    ints[0, q_len - 1, 2, 5] = bits
    print(f"[case] NaN {bits:x} {dtype} {q_len}", flush=True)
    out = paged_attention_fp4(q, kc, vc, table, [n])
    assert out[0, q_len - 1, 2].isnan().all()
    clean = out.isfinite().all(dim=-1)
    clean[0, q_len - 1, 2] = True
    assert clean.all()
