"""CPU checks of the group arrays of paged_attention_shared."""
import numpy as np
import pytest
import torch

from miniserve_amd.shared import _groups_i32

CPU = torch.device("cpu")


def test_whole_numbers_of_any_kind():
    for rows, pages in (([0, 2, 4], [3, 1]), ((0, 2, 4), (3, 1)), (np.array([0, 2, 4]), np.array([3, 1])),
                        (torch.tensor([0, 2, 4]), torch.tensor([3, 1], dtype=torch.int16)),
                        ([0.0, 2.0, 4.0], [3.0, 1.0])):
        r, p = _groups_i32(rows, pages, 4, 5, CPU)
        assert r.dtype == p.dtype == torch.int32
        assert r.tolist() == [0, 2, 4] and p.tolist() == [3, 1]


@pytest.mark.parametrize("rows,pages", [
    ([0, 2.7], [1]), ([0, 2], [1.5]), (torch.tensor([0.0, 2.0]), [1]), ([0, 2], torch.tensor([True])),
    (np.array([0.0, 1.5]), [1]),
])
def test_other_numbers_are_refused(rows, pages):
    with pytest.raises(ValueError, match="whole numbers"):
        _groups_i32(rows, pages, 4, 5, CPU)


def test_wide_values_are_the_nearest_bound():
    r, p = _groups_i32(torch.tensor([-2 ** 40, 2 ** 32 + 3]), torch.tensor([2 ** 31]), 4, 5, CPU)
    assert r.tolist() == [0, 4] and p.tolist() == [5]
