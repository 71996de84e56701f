"""The bounds that the tests of cached attention hold results to are narrow enough: results of weights rounded to bf16, formed here in 64 bits, leave those for 16 bits.  Without a GPU."""
import pytest
import torch

import cached_attention_oracle as oracle
import test_gpu_cached_attention as cases
from cached_attention_routes import prefix_is_shared


@pytest.mark.parametrize("keys,size", [(51, 64), (180, 64), (329, 64), (41, 128), (150, 128)])
def test_weights_of_8_bits_leave_the_bounds_for_16(keys, size):
    g = torch.Generator().manual_seed(keys)
    q, k, v = (torch.randn(n, size, generator=g, dtype=torch.float64).bfloat16().double() for n in (4, keys, keys))
    scale, seen = size ** -0.5, torch.ones(4, keys, dtype=torch.bool)
    want, _, off, _, mass = oracle.attention(q, k, v, seen, scale)
    p = torch.softmax(scale * (q @ k.T), 1)
    p = p / p.amax(1, keepdim=True)
    total = p.sum(1, keepdim=True)  # of the unrounded weights, as the kernels have it
    fine, coarse = ((w @ v / total).bfloat16().double() for w in (p, p.bfloat16().double()))
    for bits, coarse_fits in ((2.0 ** -8, True), (2.0 ** -16, False)):
        bound = off + mass * bits
        bound = bound + (want.abs() + bound) * 2.0 ** -8
        assert bool(((fine - want).abs() <= bound).all())
        assert bool(((coarse - want).abs() <= bound).all()) == coarse_fits


def test_which_prefixes_are_shared():
    """Long ones of more than one sequence; not those of sequences of many rows."""
    one = dict(page_size=16, kv_heads=2, head_size=64, columns=20, heads=8)
    assert prefix_is_shared(sequences=2, tokens=2, prefix=1000, **one) and prefix_is_shared(sequences=300, tokens=300, prefix=1000, **one)
    assert not prefix_is_shared(sequences=1, tokens=1, prefix=1000, **one) and not prefix_is_shared(sequences=2, tokens=2, prefix=32, **one)
    assert not prefix_is_shared(sequences=2, tokens=100, prefix=1000, **one) and not prefix_is_shared(sequences=2, tokens=2, prefix=0, **one)
    assert not any(prefix_is_shared(page, kv, size, len(s), sum(n for n, _ in s), 1 + max(-(-n // page) for _, n in s), prefix, heads)
                   for s, prefix, page, heads, kv, size in cases.SHAPES)
