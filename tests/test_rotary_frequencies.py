"""Frequencies that are mixed by pairs where the borders lie outside of the pairs; without a GPU."""
import math

import pytest
import torch

from kutacc_amd import capi


@pytest.mark.parametrize("rotated", [2, 8, 64])
@pytest.mark.parametrize("length", [0.5, 2 * math.pi, 20.0, 300.0, 4096.0, 1e6, 1e9, 1e30])
@pytest.mark.parametrize("base", [1.5, 10.0, 1e4, 1e8])
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (1.0, 0.25), (4.0, 3.99)])
def test_pairs_on_either_side_of_the_borders(rotated, length, base, fast, slow):
    """As they are for pairs that turn at least `fast` times over the length, over the factor for those that turn at most `slow` times, between the two otherwise, and no pair
    stretched less than one that turns more often.  Frequencies are formed in 64 bits and rounded once to 32."""
    factor = 16.0
    plain = base ** (-2 * torch.arange(rotated // 2, dtype=torch.float64) / rotated)
    turns = length * plain / (2 * math.pi)
    share = capi.rotary_frequencies(rotated, base=base, scaling="by_pairs", factor=factor, original_length=length, fast=fast, slow=slow).double() / plain
    near = 1e-9  # of a border: either side may be right there
    assert bool((share >= 1 / factor * (1 - 2.0 ** -23)).all()) and bool((share <= 1 + 2.0 ** -23).all())
    assert bool(((share - 1).abs() <= 2.0 ** -23)[turns >= fast * (1 + near)].all()), "fast pairs"
    assert bool(((share * factor - 1).abs() <= 2.0 ** -23)[turns <= slow * (1 - near)].all()), "slow pairs"
    assert bool((share.diff() <= 2.0 ** -22).all())


def test_a_pair_exactly_on_the_slow_border():
    assert float(capi.rotary_frequencies(8, scaling="by_pairs", factor=4.0, original_length=2 * math.pi, fast=2.0, slow=1.0)[0]) == 0.25
