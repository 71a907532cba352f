"""CPU checks of the rotated cache write: msattn_write_kv_rope, msattn_paged_attention_append_rope
and their Python callers refuse bad arguments before they launch anything, and the overlap rule of
write_kv_rope's sources."""
import ctypes

import pytest
import torch

from miniserve_amd import _native as nat, write_kv_rope
from miniserve_amd.rotary import _apart, _rows_apart, extent, rope_table

I64x3 = ctypes.c_int64 * 3


def write_args(**over):
    """Arguments of a call that would launch; device pointers are made up."""
    a = dict(query=256, qs=I64x3(2048, 1024, 64), out=4096, os=I64x3(2048, 1024, 64), k=8192,
             ks=I64x3(256, 128, 64), v=12288, vs=I64x3(256, 128, 64), kc=16384, vc=32768,
             blk=16 * 128, slot=128, head=64, table=65536, starts=65792, cos=66048, sin=131072,
             position=None, per_token=0, max_pos=100, R=64, B=2, T=2, H=4, KVH=2, D=64, bs=16,
             nb=10, W=4, st=nat.BF16, kt=nat.BF16, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("bad", [
    dict(k=None), dict(v=None), dict(ks=None), dict(vs=None), dict(kc=None), dict(vc=None),
    dict(table=None), dict(starts=None), dict(cos=None), dict(sin=None), dict(out=None),
    dict(qs=None), dict(os=None), dict(H=0), dict(KVH=0), dict(B=0), dict(T=-1), dict(D=0),
    dict(D=258, R=64), dict(R=0), dict(R=63), dict(R=66), dict(max_pos=0), dict(bs=0), dict(nb=0),
    dict(W=0), dict(st=nat.FP8_E4M3), dict(st=7), dict(kt=9), dict(k=8193), dict(v=12289),
    dict(kc=16385), dict(vc=32769), dict(query=257), dict(out=4097), dict(cos=66050),
    dict(sin=131074), dict(position=65538), dict(blk=-1), dict(slot=-1), dict(head=-1),
    dict(ks=I64x3(-1, 128, 64)), dict(vs=I64x3(256, -1, 64)), dict(qs=I64x3(2048, 1024, -64)),
    dict(os=I64x3(-2048, 1024, 64)),
], ids=lambda d: ",".join(d))
def test_write_kv_rope_refuses(bad):
    assert nat.lib().msattn_write_kv_rope(*write_args(**bad)) == nat.ERR_INVALID_ARG


def test_write_kv_rope_without_tokens_launches_nothing():
    assert nat.lib().msattn_write_kv_rope(*write_args(T=0)) == nat.OK
    assert nat.lib().msattn_write_kv_rope(*write_args(T=0, query=None, out=None, qs=None, os=None,
                                                      H=0)) == nat.OK


def append_args(**over):
    a = dict(q=256, k=512, v=768, kc=1024, vc=2048, blk=16 * 256, slot=256, head=128, table=4096,
             lens=8192, out=16384, ws=32768, ws_bytes=1 << 24, B=2, H=4, KVH=2, D=128, bs=16,
             nb=100, W=4, max_context=64, window=0, scale=0.1, qt=nat.BF16, kt=nat.BF16, cos=65536,
             sin=131072, position=None, max_pos=64, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(kc=None), 1),
    (dict(vc=None), 1), (dict(table=None), 1), (dict(lens=None), 1), (dict(out=None), 1),
    (dict(ws=None), 1), (dict(cos=None), 1), (dict(sin=None), 1), (dict(cos=65540), 1),
    (dict(sin=131080), 1), (dict(position=65538), 1), (dict(max_pos=0), 1), (dict(H=3), 1),
    (dict(D=129), 1), (dict(D=258), 1), (dict(B=0), 1), (dict(qt=nat.FP8_E4M3), 1),
    (dict(kt=5), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
    (dict(blk=-1), 1), (dict(nb=0), 1), (dict(out=16385), 1), (dict(ws=32776), 1),
    (dict(ws_bytes=256), 3), (dict(B=65536, ws_bytes=1 << 62), 2),
], ids=lambda d: ",".join(d) if isinstance(d, dict) else str(d))
def test_append_rope_refuses_before_it_writes(bad, status):
    assert nat.lib().msattn_paged_attention_append_rope(*append_args(**bad)) == status


def test_cpu_tensors_raise():
    x = torch.zeros(1, 1, 2, 8)
    c = torch.zeros(2, 16, 2, 8)
    t = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU path"):
        write_kv_rope(x, x, x, c, c, torch.zeros(1, 2), 0, t, t)


def test_rope_table_forms():
    dev = torch.device("cpu")
    t = torch.rand(5, 8)
    assert rope_table(t, dev, "cos") is t
    assert rope_table(t.double(), dev, "cos").dtype == torch.float32
    assert rope_table(torch.rand(8, 5).t(), dev, "cos").is_contiguous()
    for bad in (torch.rand(5), torch.zeros(0, 8)):
        with pytest.raises(ValueError, match="cos"):
            rope_table(bad, dev, "cos")


def test_fused_projection_views_do_not_overlap():
    qkv = torch.zeros(3, 5, 4 + 2 * 2, 8)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    assert _rows_apart(q, k) and _rows_apart(v, q) and _rows_apart(k, v)
    assert _apart(k, [q]) and _apart(q, [k, v])
    assert not _apart(qkv[:, :, 3:5], [q])        # a head in both
    assert not _apart(qkv[:, 1:], [qkv[:, :-1]])  # the same rows, a token later
    assert not _apart(q.transpose(0, 1), [k])     # other strides: not told apart
    packed = torch.zeros(2, 3, 2, 8)
    assert not _apart(packed, [packed]) and _apart(packed, [torch.zeros(2, 3, 2, 8)])
    # rows that reach into the next token's
    x = torch.zeros(64)
    assert not _rows_apart(x.as_strided((1, 2, 2, 8), (0, 8, 16, 1)),
                           x.as_strided((1, 2, 1, 8), (0, 8, 8, 1), 24))
    lo, hi = extent(q)
    assert hi - lo == (((3 - 1) * 5 + 4) * 64 + 3 * 8 + 8) * 4
    assert extent(torch.zeros(0, 3))[0] == extent(torch.zeros(0, 3))[1]
