"""CPU checks of the 4-bit cache's entry points: refusals, workspace sizes, CPU tensors."""
import pytest
import torch

from miniserve_amd import (PagedAttention, _native as nat, allocate_fp4_cache, paged_attention_fp4,
                           read_kv_fp4, write_kv_fp4)


def write_args(**over):
    a = dict(k=1 << 20, k0=768, k1=256, k2=128, v=1 << 21, v0=768, v1=256, v2=128, kc=4096, vc=1 << 17, blk=1088 * 2, head=1088, table=256,
             starts=512, B=2, T=3, KVH=2, D=128, bs=16, nb=10, W=4, t=nat.BF16, stream=None)
    a.update(over)
    return list(a.values())


BAD_CACHE = [(dict(kc=None), 1), (dict(vc=None), 1), (dict(kc=4100), 1), (dict(vc=8200), 1),
             (dict(blk=-16), 1), (dict(blk=8), 1), (dict(head=1080), 1), (dict(table=None), 1),
             (dict(table=258), 1), (dict(KVH=0), 1), (dict(D=0), 1), (dict(D=48), 1),
             (dict(D=288), 1), (dict(bs=8), 1), (dict(bs=0), 1), (dict(bs=24), 1), (dict(nb=0), 1),
             (dict(W=0), 1), (dict(B=0), 1), (dict(t=nat.FP8_E4M3), 1), (dict(t=7), 1)]


def named(d):
    return ",".join(f"{k}={v}" for k, v in d.items()) if isinstance(d, dict) else str(d)


@pytest.mark.parametrize("bad,status", BAD_CACHE + [
    (dict(k=None), 1), (dict(v=None), 1), (dict(k1=-1), 1), (dict(v0=-256), 1),
    (dict(k=4096 + 9 * 2176 + 2000), 5), (dict(v=(1 << 17) - 2 * 1536 + 16), 5), (dict(k=4096 - 100, k2=1 << 20), 5),
    (dict(starts=None), 1), (dict(starts=514), 1), (dict(k=1025), 1), (dict(T=-1), 1),
    (dict(B=1 << 20, T=1 << 15), 2)], ids=named)
def test_write_refuses(bad, status):
    assert nat.lib().msattn_write_kv_fp4(*write_args(**bad)) == status


def read_args(**over):
    a = dict(kc=4096, vc=8192, blk=1088 * 2, head=1088, table=256, starts=512, k=1024, v=2048, B=2,
             T=3, KVH=2, D=128, bs=16, nb=10, W=4, t=nat.BF16, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("bad,status", BAD_CACHE + [
    (dict(k=None), 1), (dict(v=None), 1), (dict(starts=None), 1), (dict(v=2049), 1),
    (dict(T=-1), 1), (dict(B=1 << 20, T=1 << 15), 2)], ids=named)
def test_read_refuses(bad, status):
    assert nat.lib().msattn_read_kv_fp4(*read_args(**bad)) == status


def attend_args(**over):
    a = dict(q=1024, q0=1024, q1=1024, q2=128, kc=4096, vc=8192, blk=1088 * 2, head=1088,
             table=256, lens=512, out=2048, ws=1 << 20, ws_bytes=1 << 40, B=2, q_len=1, H=8, KVH=2,
             D=128, bs=16, nb=10, W=4, max_context=64, causal=1, window=0, scale=0.1, t=nat.BF16,
             stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("bad,status", BAD_CACHE + [
    (dict(q=None), 1), (dict(q1=-1024), 1), (dict(lens=None), 1), (dict(lens=513), 1),
    (dict(out=None), 1), (dict(ws=None), 1), (dict(q=1032), 1), (dict(out=2056), 1),
    (dict(ws=(1 << 20) + 64), 1), (dict(q_len=0), 1), (dict(H=0), 1), (dict(H=3), 1),
    (dict(max_context=-1), 1), (dict(window=-1), 1), (dict(scale=float("nan")), 1),
    (dict(q0=1028), 1), (dict(q2=132), 1),
    (dict(ws_bytes=1024), 3), (dict(q_len=1 << 29), 2),
    (dict(max_context=(1 << 30) + 1), 2)], ids=named)
def test_attention_refuses(bad, status):
    assert nat.lib().msattn_paged_attention_fp4(*attend_args(**bad)) == status


def test_nothing_to_do():
    assert nat.lib().msattn_write_kv_fp4(*write_args(T=0)) == 0
    assert nat.lib().msattn_read_kv_fp4(*read_args(T=0)) == 0


def test_workspace_bytes():
    f = nat.lib().msattn_fp4_workspace_bytes
    header = (64 + 4096) * 4
    assert f(4, 1, 6, 4, 64, 100, nat.BF16) == 0 and f(4, 1, 4, 4, 48, 100, nat.BF16) == 0
    assert f(4, 1, 4, 4, 64, 100, nat.FP8_E4M3) == 0 and f(0, 1, 4, 4, 64, 100, nat.BF16) == 0
    assert f(4, 1, 4, 4, 64, 100, nat.BF16) > header
    # as many contexts as one likes need no more
    assert f(1 << 15, 1, 32, 8, 128, 1 << 16, nat.BF16) <= f(64, 1, 32, 8, 128, 1 << 16, nat.BF16)


def test_allocation():
    k, v = allocate_fp4_cache(5, 32, 3, 96, device="cpu")
    assert k.shape == v.shape == (5, 3, 2, 816) and k.dtype == torch.uint8 and not k.any()
    for bad in (dict(num_blocks=0), dict(block_size=24), dict(block_size=0), dict(num_kv_heads=0),
                dict(head_dim=80), dict(head_dim=288), dict(head_dim=0)):
        with pytest.raises(ValueError):
            allocate_fp4_cache(**{**dict(num_blocks=5, block_size=16, num_kv_heads=3, head_dim=64,
                                         device="cpu"), **bad})
    pa = PagedAttention(8, 2, 128, num_blocks=4, block_size=32, kv_dtype=torch.float4_e2m1fn_x2)
    k, v = pa.allocate_kv_cache()
    assert k.shape == v.shape == (4, 2, 2, 1088) and k.dtype == torch.uint8
    with pytest.raises(ValueError, match="tiles"):
        PagedAttention(8, 2, 128, num_blocks=4, block_size=8,
                       kv_dtype=torch.float4_e2m1fn_x2).allocate_kv_cache()


def test_cpu_tensors_raise():
    k, v = allocate_fp4_cache(5, 16, 2, 64, device="cpu")
    table = torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(1, 1, 2, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        write_kv_fp4(x, x, k, v, table)
    with pytest.raises(RuntimeError, match="no CPU path"):
        read_kv_fp4(k, v, table, 0, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_attention_fp4(x, k, v, table, [1])


def test_launches_of_too_many_threads_are_refused():
    """A wave a tile: 2^26 - 4 of them are 2^32 - 256 threads, one more a workgroup too many. Inputs
    that overlap the cache, and a workspace too small, end the calls below the limit."""
    L, most = nat.lib(), 4 * (2 ** 24 - 1)
    for KVH, B, T in ((1, most, 1), (4, most // 4, 1), (1, 1, 16 * most - 30), (4, 1, 4 * most - 15)):
        below = write_args(k=4096, B=B, KVH=KVH, T=T)
        assert L.msattn_write_kv_fp4(*below) == nat.ERR_OVERLAP, (KVH, B, T)
        above = dict(T=T + 16) if B == 1 else dict(B=B + 1)
        assert L.msattn_write_kv_fp4(*write_args(k=4096, KVH=KVH, **{**dict(B=B, T=T), **above})) == \
            nat.ERR_UNSUPPORTED, (KVH, B, T)
        assert L.msattn_read_kv_fp4(*read_args(KVH=KVH, **{**dict(B=B, T=T), **above})) == \
            nat.ERR_UNSUPPORTED, (KVH, B, T)


@pytest.mark.parametrize("KVH,H", [(8, 8), (1, 1)])
def test_attention_of_too_many_threads_is_refused(KVH, H):
    """Short contexts: whole units of eight waves, a workgroup of 512 threads each."""
    L, most = nat.lib(), (2 ** 23 - 8) // KVH
    args = dict(H=H, KVH=KVH, q_len=1, max_context=16, ws_bytes=1024)
    assert L.msattn_paged_attention_fp4(*attend_args(B=most, **args)) == nat.ERR_WORKSPACE
    for B in (most + 8, 1 << 27):
        assert L.msattn_paged_attention_fp4(*attend_args(B=B, **{**args, "ws_bytes": 1 << 40})) == \
            nat.ERR_UNSUPPORTED


@pytest.mark.parametrize("given,match", [
    (dict(shared_prefix_pages=4), "outside"), (dict(shared_prefix_pages=-1), "outside"),
    (dict(prefix_groups=([0, 3], [1])), "ascend"), (dict(prefix_groups=([1, 0], [1])), "ascend"),
    (dict(prefix_groups=([0, 2], [4])), "within"), (dict(prefix_groups=([0, 2], [1, 1])), "need"),
    (dict(prefix_groups=([0, 1.5], [1])), "whole"),
    (dict(prefix_groups=(torch.tensor([0.0, 2.0]), [1])), "whole")], ids=str)
def test_malformed_prefixes_are_refused_though_unused(given, match):
    pa = PagedAttention(4, 2, 64, num_blocks=8, block_size=16, kv_dtype=torch.float4_e2m1fn_x2)
    kc, vc = pa.allocate_kv_cache()
    q, table = torch.zeros(2, 1, 4, 64), torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match=match):
        pa(q, kc, vc, table, [1, 1], **given)
    # as over other caches, where they are not looked at: under a window, not causal, as far as the GPU
    for kw in (dict(window=5), dict(causal=False)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            pa(q, kc, vc, table, [1, 1], **given, **kw)


@pytest.mark.parametrize("given", [{}, dict(shared_prefix_pages=3), dict(shared_prefix_pages=0),
                                   dict(prefix_groups=([0, 2], [3])), dict(prefix_groups=([], []))], ids=str)
def test_prefixes_are_accepted(given):
    pa = PagedAttention(4, 2, 64, num_blocks=8, block_size=16, kv_dtype=torch.float4_e2m1fn_x2)
    kc, vc = pa.allocate_kv_cache()
    with pytest.raises(RuntimeError, match="no CPU path"):
        pa(torch.zeros(2, 1, 4, 64), kc, vc, torch.zeros(2, 3, dtype=torch.int32), [1, 1], **given)
