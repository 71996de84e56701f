"""Values near the end of fp32's range: a result that is finite comes out finite, in each form that cached attention takes."""
import pytest
import torch

from test_gpu_cached_attention import BF16, E4M3, Batch

pytestmark = pytest.mark.gpu

# (queries, length) of each sequence, and a prefix.  Few rows by eight waves, by four, their keys split; many rows, theirs split; a prefix read once for few rows and for many.
FORMS = [([(1, 700)] * 8, 0), ([(1, 700)] * 600, 0), ([(1, 1100)] * 60, 0), ([(40, 900)] * 3, 0), ([(500, 640)], 0), ([(1, 600), (1, 300)], 2000), ([(9, 600), (1, 300)], 2000)]


@pytest.mark.parametrize("dtype", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("size", [64, 256])
@pytest.mark.parametrize("sequences,prefix", FORMS)
def test_large_values_behind_growing_logits(sequences, prefix, size, dtype):
    """Logits that are 0, or 7.93 powers of two, of 32 entries at a time: less than a row's maximum is followed for.  All values of a row add up to 2^127 at most, so that no sum of them
    with weights up to one leaves fp32; with weights up to 2^7.93 it does."""
    b = Batch(sequences, prefix, 16, 1, size, dtype)
    count = prefix + max(n for _, n in sequences)
    largest = 2.0 ** 127 / count
    g = torch.Generator().manual_seed(3)
    if dtype == E4M3:
        b.scales = [torch.ones(1), torch.tensor([largest / 448])]
    for pages, n in [(b.prefix_pages, prefix)] + [(b.table[i], n) for i, (_, n) in enumerate(sequences)]:
        at = torch.arange(n)
        grows = torch.randint(0, 2, (n // 32 + 1,), generator=g).repeat_interleave(32)[:n]
        keys = (5.5 * grows)[:, None].expand(n, size).to(dtype)
        values = ((0.5 + 0.45 * torch.rand(n, size, generator=g)) * (448 if dtype == E4M3 else largest)).to(dtype)
        for cache, x in ((b.k, keys), (b.v, values)):
            cache, x = (t.view(torch.uint8) if dtype == E4M3 else t for t in (cache, x.contiguous()))
            cache[pages.long()[at // 16], at % 16, 0] = x
    out = b.check(4, scale=1.0 / size, q=torch.ones(b.tokens, 4, size, dtype=BF16), what=f"{sequences[0]} x {len(sequences)} behind {prefix}")
    assert bool(torch.isfinite(out).all())
