"""The oracle of the 4-bit cache, pinned by hand-computed answers."""
import numpy as np
import torch

from oracle import fp4


def row(*head, fill=0.0):
    return torch.tensor(list(head) + [fill] * (32 - len(head)), dtype=torch.float32)


def one(x):
    codes, scale = fp4.quantise(x)
    return fp4.values(codes, scale), scale


def test_levels_and_ties():
    # the block's largest is 6: the power is 1, and ties go to the even code
    x = row(6, 0.25, 0.2500001, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.0001, -0.0, -3.2, 1.2499999)
    v, s = one(x)
    assert s.tolist() == [127]
    assert v[:13].tolist() == [6, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 0, -3, 1]
    assert np.signbit(v[10])


def test_the_power_of_two():
    for top, byte, kept in ((4.0, 127, 4), (7.0, 127, 6), (7.0001, 128, 8), (3.5, 126, 3),
                            (3.5001, 127, 4), (1.0, 125, 1), (0.0, 1, 0)):
        v, s = one(row(top))
        assert (s.tolist(), v[0]) == ([byte], kept), top
    assert one(row(2.0 ** -140))[1].tolist() == [1]
    v, s = one(row(3.4e38))
    assert s.tolist() == [252] and v[0] == 6 * 2.0 ** 125


def test_nan_and_infinity():
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.cat((row(1.0, bad), row(1.0)))
        v, s = one(x)
        assert s.tolist() == [255, 125]
        assert np.isnan(v[:32]).all() and v[32] == 1


def test_layout():
    x = torch.randn(2, 32, 3, 64, generator=torch.Generator().manual_seed(0))
    codes, scale = fp4.quantise(x)
    for is_values in (False, True):
        c = fp4.pack(codes, scale, is_values)
        assert c.shape == (2, 3, 2, 544)
        a, b = fp4.unpack(c, is_values)
        assert (a == codes).all() and (b == scale).all()
    # token 17 (tile 1, place 1), head 2, dims 10 and 11 of page 1
    want = int(codes[1, 17, 2, 10]) | int(codes[1, 17, 2, 11]) << 4
    assert fp4.pack(codes, scale, False)[1, 2, 1, 1 * 32 + 5] == want
    assert fp4.pack(codes, scale, True)[1, 2, 1, 64 * 1 + 4 * 1 + 1] == want
    assert fp4.pack(codes, scale, True)[1, 2, 1, 512 + 16 * 1 + 1] == scale[1, 17, 2, 1]


def test_error_bound():
    x = torch.randn(500, 128, generator=torch.Generator().manual_seed(1))
    v, s = one(x)
    top = x.view(500, 4, 32).abs().amax(-1).double().numpy()
    two = 2.0 ** (s.astype(float) - 127)
    assert (top > 3.5 * two).all() and (top <= 7 * two).all()
    err = np.abs(v - x.double().numpy()).reshape(500, 4, 32).max(-1)
    assert (err <= two).all()
