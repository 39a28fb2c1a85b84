"""Sizes of the expert layer that the C arguments do not hold."""
import pytest

from bare_metal_b200 import igemm as ig


@pytest.mark.parametrize("sizes", [(2 ** 32 + 1, 64, 64, 4, 2), (2, 64, 64, 4, 2 ** 32 + 2), (2, 2 ** 32 + 64, 64, 4, 2), (2, 64, 2 ** 32 + 64, 4, 2),
                                   (2, 64, 64, 2 ** 32 + 4, 2), (-2 ** 32 + 1, 64, 64, 4, 2), (65, 64, 64, 4, 2), (2, 64, 64, 4, 5), (0, 64, 64, 4, 2)])
def test_a_size_beyond_an_int_does_not_come_back_as_a_small_one(sizes):
    with pytest.raises(ig.BmError):
        ig._moe_f4_bytes(*sizes)


def test_sizes_that_are_allowed():
    assert ig._moe_f4_bytes(64, 16384, 16384, 256, 16) > ig._moe_f4_bytes(1, 1, 1, 1, 1) > 0
