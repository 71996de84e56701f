"""Calls of cached attention, the append and rotary positions that are allowed and rare: other orders of a cache's axes, page tables without columns, more tokens than a launch has
workgroups, what an 8-bit cache holds where nobody looks."""
import math

import pytest
import torch

import cached_attention_oracle as oracle
from kutacc_amd import capi
from test_gpu_cached_attention import BF16, E4M3, FILL, INT32, Batch, ok, randn

pytestmark = pytest.mark.gpu


class Ordered(Batch):
    """With its cache's axes (pages, slots, heads) stored in another order, the outermost first."""

    order = (0, 1, 2)

    def _on_gpu(self, x):
        back = [self.order.index(i) for i in range(3)]
        return x.permute(*self.order, 3).contiguous().cuda().permute(*back, 3)


@pytest.mark.parametrize("dtype", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("order", [(0, 2, 1), (1, 0, 2), (1, 2, 0), (2, 0, 1), (2, 1, 0)])
@pytest.mark.parametrize("page", [16, 5])
def test_a_cache_in_any_order(page, order, dtype):
    for sequences, prefix, heads in (([(1, 40), (1, 300)], 50, 8), ([(40, 40), (3, 200)], 0, 4), ([(1, 40), (9, 90)], 1030, 8)):
        b = Ordered(sequences, prefix, page, 2, 64, dtype, seed=page)
        b.order = order
        b.check(heads, what=f"{order} {prefix}")
    k = randn(3, b.tokens, 2, 64)
    ok(capi.CacheAppend(b.cache, b.batch, k.cuda(), k.cuda()))
    for i, (n, length) in enumerate(b.sequences):
        for j in range(n):
            at = length - n + j
            for got, scales in zip(b.gpu, b.scales):
                want = oracle.d(k[b.starts[i] + j]) / (1.0 if scales is None else oracle.d(scales)[:, None])
                oracle.close(got[int(b.table[i, at // page]), at % page], want, oracle.stored(want, want.abs() * 2.0 ** -24, dtype), f"{order} entry {at}")


@pytest.mark.parametrize("prefix", [1, 40, 700, 1024, 1031])
@pytest.mark.parametrize("queries", [1, 20])
def test_a_page_table_without_columns(queries, prefix):
    """Sequences that have nothing but the prefix, whatever their lengths say."""
    b = Batch([(queries, 0), (2, 0), (0, 0)], prefix, 16, 2, 64, spare_columns=0, seed=prefix)
    assert b.table.shape[1] == 0
    b.check(4, what="of length 0")
    b.lengths[:2] = torch.tensor([queries + 3, 1], dtype=INT32)
    b.sequences = [(queries, queries + 3), (2, 1), (0, 0)]
    b.check(4, what="of entries that are nowhere")
    cache, batch = b.on_gpu()
    before = b.gpu[0].clone()
    k = randn(1, b.tokens, 2, 64).cuda()
    ok(capi.CacheAppend(cache, batch, k, k))
    assert torch.equal(b.gpu[0].view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("page", [16, 6])
@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("heads,queries", [(2, 7), (2, 60), (16, 33)])
@pytest.mark.parametrize("prefix", [0, 40])
def test_what_is_not_seen_of_an_8_bit_cache_may_be_anything(prefix, heads, queries, size, page):
    """NaN among the entries that a token must not see yet changes no bit of its results; in one that it sees, of its own."""
    b = Batch([(queries, queries + 10), (5, 90)], prefix, page, 1, size, E4M3, seed=5)
    q = randn(9, b.tokens, heads, size).cuda()
    cache, batch = b.on_gpu()
    clean, out = torch.empty_like(q), torch.empty_like(q)
    ok(capi.CachedAttention(cache, batch, q, clean))
    entry = queries + 5  # of the first sequence: seen by its last five tokens
    place = int(b.table[0, entry // page]), entry % page
    b.gpu[1].view(torch.uint8)[place[0], place[1], 0, 2] = 0x7f
    ok(capi.CachedAttention(cache, batch, q, out))
    sees = [i for i in range(queries) if 10 + i >= entry]
    rest = [i for i in range(b.tokens) if i not in sees]
    assert len(sees) == 5 and torch.equal(out[rest].view(torch.int16), clean[rest].view(torch.int16))
    assert bool(torch.isnan(out[sees][..., 2]).all())
    others = [c for c in range(size) if c != 2]
    assert bool(torch.isfinite(out[sees][..., others]).all())
    b.gpu[0].view(torch.uint8)[place[0], place[1], 0, 7] = 0xff
    ok(capi.CachedAttention(cache, batch, q, out))
    assert torch.equal(out[rest].view(torch.int16), clean[rest].view(torch.int16)) and bool(torch.isnan(out[sees]).all())


def test_rotary_of_more_tokens_than_a_launch_has_places_for():
    tokens = (1 << 19) + 12345
    x, inv_freq = randn(1, tokens, 1, 4), capi.rotary_frequencies(4)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(2), dtype=INT32)
    out = torch.full((tokens + 3, 1, 4), FILL, dtype=BF16, device="cuda")
    ok(capi.Rotary(x.cuda(), inv_freq.cuda(), positions.cuda(), q_out=out[:tokens]))
    want, off = oracle.rotated(x, positions, inv_freq)
    oracle.close(out[:tokens], want, oracle.stored(want, off, BF16), "far tokens")
    assert bool((out[tokens:] == FILL).all())


def test_append_of_more_tokens_than_a_launch_has_places_for():
    page, counts = 64, [(1 << 19) + 77, 0, 4000]
    pages = [-(-n // page) for n in counts]
    tokens, size = sum(counts), 16
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(1)).to(INT32)
    table = torch.full((3, max(pages)), -1, dtype=INT32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0, counts[0], counts[0], tokens], dtype=INT32)
    caches = [torch.full((sum(pages), page, 1, size), math.nan, dtype=BF16, device="cuda") for _ in range(2)]
    k, v = randn(1, tokens, 1, size), randn(2, tokens, 1, size)
    ok(capi.CacheAppend(capi.Cache(*caches), capi.CacheBatch(starts.cuda(), torch.tensor(counts, dtype=INT32).cuda(), table.cuda()), k.cuda(), v.cuda()))
    for x, cache in ((k, caches[0]), (v, caches[1])):
        cache = cache.cpu()
        for i in (0, 2):
            entry = torch.arange(counts[i])
            assert torch.equal(cache[table[i].long()[entry // page], entry % page], x[int(starts[i]):int(starts[i + 1])])
        assert int(torch.isnan(cache).all(3).sum()) == sum(pages) * page - tokens
