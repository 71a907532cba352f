"""CPU checks of msattn_paged_attention_shared's refusals and of its workspace size."""
import pytest

from miniserve_amd import _native as nat


def args(**over):
    a = dict(q=256, kc=1024, vc=2048, blk=16 * 256, slot=256, head=128, table=4096, lens=8192,
             rows=8448, pages=8704, groups=2, out=16384, ws=32768, ws_bytes=1 << 40, B=4, q_len=1,
             H=4, KVH=2, D=128, bs=16, nb=100, W=4, max_context=64, scale=0.1, qt=nat.BF16,
             kt=nat.BF16, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("bad,status", [
    (dict(q=None), 1), (dict(kc=None), 1), (dict(vc=None), 1), (dict(table=None), 1),
    (dict(lens=None), 1), (dict(rows=None), 1), (dict(pages=None), 1), (dict(out=None), 1),
    (dict(ws=None), 1), (dict(groups=-1), 1), (dict(B=0), 1), (dict(q_len=0), 1), (dict(H=3), 1),
    (dict(D=129), 1), (dict(D=258), 1), (dict(max_context=-1), 1), (dict(bs=0), 1), (dict(nb=0), 1),
    (dict(W=0), 1), (dict(blk=-1), 1), (dict(slot=-2), 1), (dict(head=-1), 1),
    (dict(scale=float("nan")), 1), (dict(qt=nat.FP8_E4M3), 1), (dict(kt=9), 1), (dict(q=257), 1),
    (dict(out=16385), 1), (dict(ws=32776), 1), (dict(rows=8450), 1), (dict(pages=8705), 1),
    (dict(ws_bytes=1024), 3),
], ids=lambda d: ",".join(d) if isinstance(d, dict) else str(d))
def test_refuses(bad, status):
    assert nat.lib().msattn_paged_attention_shared(*args(**bad)) == status


def test_workspace_bytes():
    f = nat.lib().msattn_shared_workspace_bytes
    base = nat.lib().msattn_workspace_bytes
    assert f(4, 1, 6, 4, 64, 100, 1) == 0 and f(4, 1, 4, 4, 64, 100, -1) == 0
    # no group, or a geometry the kernel leaves to the others: their workspace
    assert f(4, 1, 4, 4, 64, 100, 0) == base(4, 1, 4, 4, 64, 100)
    assert f(2000, 1, 4, 4, 64, 100, 3) == base(2000, 1, 4, 4, 64, 100)
    assert f(4, 1, 4, 4, 80, 100, 3) == base(4, 1, 4, 4, 80, 100)
    # the header other calls keep their counters in, the plan (8 words a row), then two partial
    # rows an output row and 128 a share of 256: (m, l) and an accumulator each
    r256 = lambda x: -(-x // 256) * 256  # noqa: E731
    slots = 2 * 64 * 32 + 256 * 128
    want = r256(4 * (64 + 4096)) + r256(4 * (16 + 8 * 64)) + r256(8 * slots) + \
        slots * 128 * 4
    assert f(64, 1, 32, 8, 128, 1024, 8) == max(want, base(64, 1, 32, 8, 128, 1024))
