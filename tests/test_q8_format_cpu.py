"""What a growing scale does to the values that a page holds."""

import torch

from tests import plain_q8 as plain

F8 = torch.float8_e4m3fn


def test_a_growing_scale_rounds_again_below_2_to_the_minus_6_alone():
    held = torch.arange(256, dtype=torch.uint8).view(F8).double()
    held = held[~held.isnan()]
    for k in range(1, 30):
        moved = held * 2.0 ** -k                                   # in units of a scale 2^k as large
        again = plain.e4m3(moved)
        small = moved.abs() < 2.0 ** -6
        assert torch.equal(again[~small], moved[~small])
        assert float((again - moved).abs().max()) <= 2.0 ** -10
    # by all of that where it falls in the middle
    assert float((plain.e4m3(torch.tensor([2.0 ** -9 * 1.5, 2.0 ** -10], dtype=torch.float64)) - torch.tensor([2.0 ** -9 * 1.5, 2.0 ** -10])).abs().max()) == 2.0 ** -10


def test_a_pages_largest_value_is_above_224_scales():
    for top in torch.logspace(-12, 14, 4000, dtype=torch.float64).tolist():
        s = plain.scale_for(top)
        assert 224 * s < top <= 448 * s or s == 2.0 ** -50
