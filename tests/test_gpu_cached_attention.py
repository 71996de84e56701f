"""Rotary positions, the cache in pages and the attention over it on the GPU, against their definitions in 64 bits."""
import math

import pytest
import torch

import cached_attention_oracle as oracle
from kutacc_amd import capi

pytestmark = pytest.mark.gpu

BF16, FP32, E4M3, INT32 = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.int32
FILL = 77.0  # what surrounds a result and has to stay


def randn(seed, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def ok(call):
    rc = call.run()
    torch.cuda.synchronize()
    assert rc == 0, rc


class Placed:
    """A [tokens, heads, size] tensor inside a larger one that has to keep what is around it: `pad` channels behind a head, `offset` elements in front, heads outside
    of the tokens with `outer`."""

    def __init__(self, tokens, heads, size, dtype=BF16, pad=0, offset=0, outer=False, values=None):
        shape = (heads, tokens, size + pad) if outer else (tokens, heads, size + pad)
        self.buffer = torch.full((offset + math.prod(shape) + 5,), FILL, dtype=FP32).to(dtype).cuda()
        whole = self.buffer[offset:offset + math.prod(shape)].view(shape)
        self.view = (whole.transpose(0, 1) if outer else whole)[..., :size]
        self.mask = torch.zeros_like(self.buffer, dtype=torch.bool)
        mask = self.mask[offset:offset + math.prod(shape)].view(shape)
        (mask.transpose(0, 1) if outer else mask)[..., :size] = True
        if values is not None:
            self.view.copy_(values.cuda())

    def untouched(self, what):
        around = self.buffer.float()[~self.mask]
        assert bool((around == FILL).all()), f"{what}: written outside of its channels"


# ---- rotary positions ----

ROTARY = [  # tokens, q heads, k heads, size, rotated, first, interleaved
    (1, 1, 0, 2, 2, 0, False), (1, 32, 8, 128, 128, 0, False), (3, 4, 4, 64, 64, 0, True), (17, 3, 1, 96, 64, 0, False), (16, 5, 5, 80, 40, 40, False),
    (33, 2, 7, 48, 24, 8, True), (5, 3, 2, 37, 20, 11, False), (5, 3, 2, 37, 36, 1, True), (100, 1, 1, 256, 256, 0, False), (2, 6, 3, 300, 128, 100, True),
    (9, 3, 2, 512, 512, 0, False), (8, 2, 2, 64, 0, 0, False), (2100, 4, 2, 64, 64, 0, False), (4099, 3, 1, 32, 32, 0, True), (300, 40, 8, 128, 128, 0, False), (7, 2, 2, 12, 8, 4, False),
]


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("tokens,heads,k_heads,size,turned,first,interleaved", ROTARY)
def test_rotary(tokens, heads, k_heads, size, turned, first, interleaved, dtype):
    inverse, magnitude, odd = tokens % 2 == 0, 1.0 if tokens % 3 else 1.2079, tokens % 5 == 1
    q, k = randn(1, tokens, heads, size, dtype=dtype), randn(2, tokens, max(k_heads, 1), size, dtype=dtype)
    inv_freq = 10000.0 ** -(torch.arange(turned // 2, dtype=FP32) / max(turned // 2, 1))
    positions = torch.randint(-5, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(3), dtype=INT32)
    qi, ki = Placed(tokens, heads, size, dtype, pad=3 * odd, offset=odd, values=q), Placed(tokens, max(k_heads, 1), size, dtype, outer=odd, values=k)
    qo, ko = Placed(tokens, heads, size, dtype, pad=8, outer=not odd), Placed(tokens, max(k_heads, 1), size, dtype, pad=odd, offset=3 * odd)
    more = dict(k=ki.view, k_out=ko.view) if k_heads else {}
    ok(capi.Rotary(qi.view, inv_freq.cuda(), positions.cuda(), q_out=qo.view, interleaved=interleaved, first=first, magnitude=magnitude, inverse=inverse, **more))
    magnitude = float(torch.tensor(magnitude))
    for x, o, what in ((q, qo, "q"), (k, ko, "k")):
        if what == "k" and not k_heads:
            continue
        want, off = oracle.rotated(x, positions, inv_freq, interleaved, first, inverse, magnitude)
        oracle.close(o.view, want, oracle.stored(want, off, dtype), what)
        outside = torch.ones(size, dtype=torch.bool)
        outside[first:first + turned] = False
        assert torch.equal(o.view.cpu()[..., outside], x[..., outside]), f"{what}: channels that are not turned"
        o.untouched(what)


def test_rotary_in_place_and_by_index():
    q = randn(4, 50, 6, 64)
    inv_freq = capi.rotary_frequencies(64, 500000.0)
    there = q.cuda()
    ok(capi.Rotary(there, inv_freq.cuda()))
    want, off = oracle.rotated(q, torch.arange(50), inv_freq)
    oracle.close(there, want, oracle.stored(want, off, BF16), "in place")
    back = capi.Rotary(there, inv_freq.cuda(), inverse=True)
    ok(back)
    oracle.close(there, oracle.d(q), 3 * 2.0 ** -8 * (oracle.d(q).abs() + oracle.d(q).roll(32, 2).abs()), "and back")


def test_rotary_gradient():
    """The rotation with `inverse` is the gradient of the one without: against the formula's by autograd in 64 bits, and against differences of the call itself."""
    x, dy = randn(5, 3, 2, 16, dtype=FP32), randn(6, 3, 2, 16, dtype=FP32)
    inv_freq, positions, m = capi.rotary_frequencies(12), torch.tensor([3, 700, 100000], dtype=INT32), 1.25
    for interleaved in (False, True):
        leaf = x.double().requires_grad_()
        a, b = (leaf[..., 2:14:2], leaf[..., 3:14:2]) if interleaved else (leaf[..., 2:8], leaf[..., 8:14])
        angle = (positions.double()[:, None] * inv_freq.double())[:, None]
        c, s = m * torch.cos(angle), m * torch.sin(angle)
        one, two = a * c - b * s, b * c + a * s
        turned = torch.stack([one, two], -1).flatten(2) if interleaved else torch.cat([one, two], -1)
        y = torch.cat([leaf[..., :2], turned, leaf[..., 14:]], -1)
        y.backward(dy.double())
        grad = torch.empty_like(x).cuda()
        ok(capi.Rotary(dy.cuda(), inv_freq.cuda(), positions.cuda(), q_out=grad, interleaved=interleaved, first=2, magnitude=m, inverse=True))
        want, off = oracle.rotated(dy, positions, inv_freq, interleaved, 2, True, m)
        assert torch.allclose(want, leaf.grad, rtol=1e-12, atol=1e-12)
        oracle.close(grad, leaf.grad, oracle.stored(leaf.grad, off, FP32), "gradient")

        def run(at):
            out = torch.empty_like(x).cuda()
            ok(capi.Rotary(at.float().cuda(), inv_freq.cuda(), positions.cuda(), q_out=out, interleaved=interleaved, first=2, magnitude=m))
            return float((out.cpu().double() * dy.double()).sum())
        for at in ((0, 0, 0), (1, 1, 5), (2, 0, 13)):
            step = torch.zeros_like(x)
            step[at] = 1.0  # linear: the difference is exact but for the roundings of some 100 products of about 1
            assert abs((run(x + step) - run(x - step)) / 2.0 - float(leaf.grad[at])) < 200 * 4 * 2.0 ** -22


# ---- the cache ----

class Batch:
    """Sequences of (queries, length), a prefix, and a cache with their pages in no order; what belongs to nobody holds NaN.  lengths may lie about what is there."""

    def __init__(self, sequences, prefix, page, kv_heads, size, dtype=BF16, seed=0, layout="slots", in_front=0, behind=0, spare_columns=1, values=None):
        self.sequences, self.prefix, self.page, self.kv_heads, self.size, self.dtype = sequences, prefix, page, kv_heads, size, dtype
        g = torch.Generator().manual_seed(seed)
        counts = [-(-max(n, 0) // page) for _, n in sequences]
        shared = -(-prefix // page)
        self.pages = shared + sum(counts) + 2
        order = torch.randperm(self.pages, generator=g)
        self.prefix_pages = order[:shared].to(INT32)
        self.columns = max(counts + [0]) + spare_columns
        self.table = torch.full((len(sequences), self.columns), -7, dtype=INT32)
        at = shared
        for i, n in enumerate(counts):
            self.table[i, :n] = order[at:at + n].to(INT32)
            at += n
        starts = [in_front]
        for n, _ in sequences:
            starts.append(starts[-1] + n)
        self.starts, self.tokens = starts, starts[-1] + behind
        self.query_starts, self.lengths = torch.tensor(starts, dtype=INT32), torch.tensor([n for _, n in sequences], dtype=INT32)
        self.scales = [None, None]
        if dtype == E4M3:
            self.scales = [0.01 + 0.02 * torch.rand(kv_heads, generator=g) for _ in range(2)]
        self.k, self.v = (self._filled(g, s, values) for s in self.scales)
        self.layout = layout

    def _filled(self, g, scales, values):
        """Numbers where somebody's entries are, NaN elsewhere."""
        x = torch.randn(self.pages, self.page, self.kv_heads, self.size, generator=g)
        if values is not None:
            x = values(x)
        if scales is not None:
            x = (x / scales[:, None]).clamp(-448, 448)
        x = x.to(self.dtype)
        mine = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for pages, count in [(self.prefix_pages, self.prefix)] + [(self.table[i], max(n, 0)) for i, (_, n) in enumerate(self.sequences)]:
            at = torch.arange(count)
            mine[pages.long()[at // self.page], at % self.page] = True
        raw = x.view(torch.uint8) if self.dtype == E4M3 else x
        raw[~mine] = 0x7f if self.dtype == E4M3 else math.nan
        return x

    def _on_gpu(self, x):
        if self.layout == "heads":  # [pages, kv_heads, page_size, size], as a view
            return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        if self.layout == "padded":
            whole = torch.empty(self.pages, self.page + 1, self.kv_heads, self.size + 32, dtype=self.dtype, device="cuda")
            (whole.view(torch.uint8) if self.dtype == E4M3 else whole).fill_(0x7f if self.dtype == E4M3 else math.nan)
            view = whole[:, :self.page, :, :self.size]
            view.copy_(x.cuda())
            return view
        return x.cuda()

    def on_gpu(self):
        self.gpu = [self._on_gpu(x) for x in (self.k, self.v)]
        self.cache = capi.Cache(*self.gpu, *(None if s is None else s.cuda() for s in self.scales))
        self.batch = capi.CacheBatch(self.query_starts.cuda(), self.lengths.cuda(), self.table.cuda(), self.prefix_pages.cuda() if self.prefix else None, self.prefix)
        return self.cache, self.batch

    def coarse(self, group):
        """Of the weights: what their rounding is relative to the weight.  16 bits of them are kept in tiles of up to 16 rows."""
        average = -(-self.tokens * group // min(len(self.sequences), self.tokens))
        whole_batch = self.prefix > 0 and len(self.sequences) > 1 and average <= 64
        return 2.0 ** -16 if average <= 16 and (not whole_batch or self.tokens * group <= 16) else 2.0 ** -8

    def attention(self, q, scale, causal):
        """Results, lse, and bounds, rows of padding as NaN."""
        heads = q.shape[1]
        group = heads // self.kv_heads
        out, bound = (torch.full(q.shape, math.nan, dtype=torch.float64) for _ in range(2))
        lse, lse_bound = (torch.full(q.shape[:2], math.nan, dtype=torch.float64) for _ in range(2))
        shared = [oracle.placed(x, s, self.prefix_pages.tolist(), self.page, self.prefix) for x, s in zip((self.k, self.v), self.scales)]
        for i, (n, length) in enumerate(self.sequences):
            own_count = min(max(length, 0), self.columns * self.page)
            own = [oracle.placed(x, s, self.table[i].tolist(), self.page, own_count) for x, s in zip((self.k, self.v), self.scales)]
            k, v = (torch.cat([a[0], b[0]]) for a, b in zip(shared, own))
            there = torch.cat([shared[0][1], own[0][1]])
            k, v = torch.where(there[:, None, None], k, torch.zeros_like(k)), torch.where(there[:, None, None], v, torch.zeros_like(v))
            at = torch.cat([torch.full((self.prefix,), -10 ** 9), torch.arange(own_count)])
            query = max(length, 0) - n + torch.arange(n)
            seen = there[None] & ((at[None] <= query[:, None]) if causal else torch.ones(n, 1, dtype=torch.bool))
            rows = slice(self.starts[i], self.starts[i] + n)
            for h in range(heads):
                o, e, off, e_off, mass = oracle.attention(q[rows, h].double(), k[:, h // group], v[:, h // group], seen, scale)
                out[rows, h], lse[rows, h], lse_bound[rows, h] = o, e, e_off
                bound[rows, h] = off + mass * self.coarse(group)
        return out, lse, bound + (out.abs() + bound) * 2.0 ** -8, lse_bound

    def check(self, heads, causal=True, scale=None, seed=9, q=None, pad=0, offset=0, outer=False, what=""):
        q = randn(seed, self.tokens, heads, self.size) if q is None else q
        scale = self.size ** -0.5 if scale is None else scale
        cache, batch = self.on_gpu()
        qi, out = Placed(self.tokens, heads, self.size, pad=pad, offset=offset, outer=outer, values=q), Placed(self.tokens, heads, self.size, pad=pad, offset=offset, outer=not outer)
        lse = torch.full((self.tokens, heads), FILL, device="cuda")
        call = capi.CachedAttention(cache, batch, qi.view, out.view, scale=scale, causal=causal, lse=lse)
        call.workspace.fill_(0xff)  # NaN: nothing of it is taken for written
        ok(call)
        want, want_lse, bound, lse_bound = self.attention(q, float(torch.tensor(scale)), causal)
        mine = slice(self.starts[0], self.starts[-1])
        oracle.close(out.view[mine], want[mine], bound[mine], f"out {what}")
        oracle.close(lse[mine], want_lse[mine], lse_bound[mine], f"lse {what}")
        for t in (out.view, lse):
            assert bool((t[:mine.start] == FILL).all()) and bool((t[mine.stop:] == FILL).all()), f"{what}: rows of padding"
        out.untouched(what)
        first = out.buffer.clone()
        call.workspace.fill_(0xff)
        ok(call)
        assert torch.equal(first.view(torch.int16), out.buffer.view(torch.int16)), f"{what}: other bits the second time"
        bits = out.view.contiguous().clone()
        out.buffer.fill_(FILL)
        ok(capi.CachedAttention(cache, batch, qi.view, out.view, scale=scale, causal=causal))
        assert torch.equal(bits.view(torch.int16), out.view.contiguous().view(torch.int16)), f"{what}: other bits without lse"
        return out.view


SHAPES = [  # (queries, length) of each sequence, prefix, page, heads, kv_heads, size
    ([(1, 1)], 0, 1, 1, 1, 8),
    ([(1, 1)], 0, 16, 32, 8, 128),
    ([(1, 31), (1, 32), (1, 33), (1, 0), (1, 127), (1, 128), (1, 129), (1, 1000)], 0, 16, 8, 2, 128),
    ([(1, 5), (1, 500)], 0, 3, 4, 4, 64),
    ([(1, 700), (0, 50), (1, 2)], 0, 64, 5, 1, 72),
    ([(1, 257), (1, 64)], 0, 7, 16, 2, 256),
    ([(1, 90)], 300, 16, 8, 8, 16),
    ([(1, 4000)], 0, 16, 8, 1, 128),
    ([(1, 9), (1, 33), (1, 200)], 100, 16, 8, 2, 128),
    ([(1, 0), (1, 1), (1, 0)], 129, 32, 16, 4, 64),
    ([(4, 30), (4, 100), (3, 3)], 77, 16, 4, 4, 64),
    ([(1, 40)] * 40, 520, 16, 8, 2, 128),
    ([(2, 40)] * 33, 1, 5, 6, 2, 192),
    ([(5, 40), (1, 1), (7, 300)], 0, 16, 7, 1, 128),
    ([(20, 20), (33, 100)], 0, 16, 4, 2, 64),
    ([(40, 64), (17, 17)], 50, 16, 2, 1, 128),
    ([(100, 100)], 0, 64, 4, 1, 128),
    ([(129, 129), (1, 1), (65, 200)], 0, 16, 2, 2, 128),
    ([(130, 400), (200, 200)], 333, 32, 4, 2, 128),
    ([(300, 300)], 0, 16, 8, 8, 64),
    ([(70, 90), (3, 3)], 40, 16, 6, 2, 256),
    ([(9, 5), (3, 0), (2, 1)], 0, 16, 2, 1, 128),
    ([(9, 5), (3, 0), (2, 1), (300, 100)], 33, 16, 2, 1, 64),
    ([(1, 1 + 7 * i % 90) for i in range(300)], 40, 16, 64, 8, 16),
    ([(1, 1 + 7 * i % 90) for i in range(300)], 0, 16, 64, 8, 16),
    ([(12, 20 + i) for i in range(100)], 70, 16, 10, 2, 32),
    ([(1, 7 * i % 300) for i in range(70)], 0, 16, 4, 2, 128),
]


@pytest.mark.parametrize("dtype", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("sequences,prefix,page,heads,kv_heads,size", SHAPES)
def test_attention(sequences, prefix, page, heads, kv_heads, size, causal, dtype):
    if dtype == E4M3 and size % 16:
        pytest.skip("no whole pieces of 16 bytes")
    odd = len(sequences) % 2
    layout = ("slots", "heads", "padded")[(page + len(sequences)) % 3]
    b = Batch(sequences, prefix, page, kv_heads, size, dtype, layout=layout, in_front=odd * 2, behind=3 - odd)
    b.check(heads, causal, pad=3 * odd, offset=odd, outer=page % 2 == 0, what=f"{sequences} {prefix} {page} {heads} {kv_heads} {size}")


def test_attention_lengths_around_every_border():
    """One sequence after the other, of lengths around the tiles', the blocks' and the pages' ends, with a few tokens each."""
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 511, 512, 513, 1023, 1025]
    for page in (16, 48, 20):
        for size, heads, kv_heads, tokens in ((128, 4, 2, 1), (64, 3, 1, 5), (128, 40, 1, 3)):
            b = Batch([(min(tokens, n), n) for n in lengths], 0, page, kv_heads, size, seed=page, spare_columns=0)
            b.check(heads, what=f"{page} {size} {tokens}")


@pytest.mark.parametrize("queries", [1, 3, 40])
def test_prefix_lengths_around_every_border(queries):
    for prefix in (1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 1000, 1024, 1025):
        b = Batch([(queries, 50), (queries, 41), (queries, 300)], prefix, 16, 2, 64, seed=prefix)
        b.check(4, what=f"{queries} {prefix}")


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("size", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [16, 6])
def test_prefixes_that_are_read_once(page, size, cache):
    """Long ones, and short ones of many sequences: a batch of 16 rows and less, and more, of each sequence up to 16 and more; a page of the prefix that is not there."""
    for prefix, spans, heads, kv_heads in ((769, [(1, 50), (1, 1)], 8, 1), (800, [(1, 300), (0, 9), (3, 41), (1, 700)], 4, 2), (1030, [(8, 20), (16, 300), (5, 5)], 4, 1),
                                           (77, [(1, 1 + i % 90) for i in range(3500)], 1, 1)):
        b = Batch(spans, prefix, page, kv_heads, size, cache, seed=prefix)
        b.prefix_pages[prefix // page // 2] = -1
        b.check(heads, what=f"{prefix} {len(spans)}")


@pytest.mark.parametrize("queries,prefix", [(1, 0), (1, 70), (30, 0), (30, 70), (200, 70)])
def test_pages_that_are_not_there(queries, prefix):
    """Their entries are not seen, whatever number stands for them."""
    b = Batch([(queries, 200), (queries, 333), (min(queries, 16), 16), (queries, 210)], prefix, 16, 2, 64, seed=3)
    b.table[0, 2], b.table[0, 5], b.table[1, 0], b.table[1, -2], b.table[2, 0] = -1, b.pages, -(1 << 31), (1 << 31) - 1, -5
    if prefix:
        b.prefix_pages[1] = b.pages + 7
    b.check(4, what="missing pages")


def test_a_length_past_the_page_table():
    """Entries past its columns are not there; positions are those of the length all the same."""
    b = Batch([(4, 100), (1, 64), (4, -3)], 30, 16, 2, 64, spare_columns=0)
    b.lengths[0], b.lengths[1] = 130, 1000
    b.sequences = [(4, 130), (1, 1000), (4, -3)]
    b.check(4, what="past the table")


@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("heads,queries", [(2, 7), (2, 60), (16, 33)])
@pytest.mark.parametrize("page", [16, 6])
def test_what_is_not_seen_may_be_anything(heads, queries, size, page):
    """Infinities and NaN among the entries that a token must not see yet change nothing of its results; those of the tokens that see them are theirs."""
    b = Batch([(queries, queries + 10), (5, 90)], 0, page, 1, size, seed=5)
    q = randn(9, b.tokens, heads, size)
    cache, batch = b.on_gpu()
    clean, out = torch.empty(b.tokens, heads, size, dtype=BF16, device="cuda"), torch.empty(b.tokens, heads, size, dtype=BF16, device="cuda")
    ok(capi.CachedAttention(cache, batch, q.cuda(), clean))
    wild = {(0, queries + 4): (math.nan, math.inf), (0, queries + 8): (1.0, -math.inf), (1, 88): (math.inf, math.nan)}  # (sequence, entry): of its key, of its value
    for (s, at), (k, v) in wild.items():
        page_at = int(b.table[s, at // page])
        b.gpu[0][page_at, at % page, 0, 3], b.gpu[1][page_at, at % page, 0, 1] = k, v
    ok(capi.CachedAttention(cache, batch, q.cuda(), out))
    first = queries + 10 - queries  # entries in front of the first token's
    free = list(range(0, queries + 4 - first)) + list(range(queries, queries + 3))  # tokens that see none of them
    assert torch.equal(out[free].view(torch.int16), clean[free].view(torch.int16))
    seen = [queries + 4 - first, queries - 1, queries + 3, queries + 4]
    assert bool(torch.isnan(out[seen]).any(2).all()), "a NaN that is seen"
    # values alone: an infinity stays one, in its channel alone
    b2 = Batch([(queries, queries + 10)], 0, page, 1, size, seed=5)
    cache, batch = b2.on_gpu()
    at = queries + 6
    b2.gpu[1][int(b2.table[0, at // page]), at % page, 0, 2] = -math.inf
    q = randn(9, b2.tokens, heads, size)
    ok(capi.CachedAttention(cache, batch, q.cuda(), out[:queries]))
    sees = torch.arange(queries) + 10 >= at
    assert bool((out[:queries][sees][..., 2] == -math.inf).all()) and bool(torch.isfinite(out[:queries][~sees]).all())
    rest = out[:queries].clone()
    rest[..., 2] = 0
    assert bool(torch.isfinite(rest).all())


@pytest.mark.parametrize("some,count", [(10, 200), (60, 64), (64, 65), (65, 65), (90, 150), (150, 150)])
def test_many_sequences_whose_keys_are_split(some, count):
    """More sequences than a wave has lanes, some of them without tokens, lengths around 2500 among short ones: shares that stay in a tile and such that go over its end."""
    g = torch.Generator().manual_seed(some)
    lengths = torch.where(torch.rand(count, generator=g) < 0.1, 2400 + torch.randint(0, 200, (count,), generator=g), torch.randint(1, 90, (count,), generator=g)).tolist()
    lengths[-1] = lengths[0] = 2600
    with_tokens = {0, count - 1, *torch.randperm(count, generator=g)[:some - 2].tolist()}
    spans = [(int(i in with_tokens), n) for i, n in enumerate(lengths)]
    for prefix in (0, 100):
        Batch(spans, prefix, 16, 1, 64, seed=1).check(4, what=f"{some} of {count}, prefix {prefix}")


@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("heads,queries,length", [(2, 1, 150), (4, 1, 3000), (4, 40, 700)])
def test_an_infinite_value_that_all_see_stays_one(size, heads, queries, length):
    """Far in front of every token's end, with a weight that is not zero: infinite in its channel, and nothing changes in the others."""
    b = Batch([(queries, length)] * 2, 0, 16, 1, size, seed=5)
    q = randn(9, b.tokens, heads, size)
    cache, batch = b.on_gpu()
    clean, out = (torch.empty(b.tokens, heads, size, dtype=BF16, device="cuda") for _ in range(2))
    ok(capi.CachedAttention(cache, batch, q.cuda(), clean))
    for at, channel, value in ((3, 0, math.inf), (40, 5, -math.inf), (97, size - 1, math.inf)):
        b.gpu[1][int(b.table[0, at // 16]), at % 16, 0, channel] = value
    ok(capi.CachedAttention(cache, batch, q.cuda(), out))
    got = out[:queries]
    assert bool((got[..., 0] == math.inf).all()) and bool((got[..., 5] == -math.inf).all()) and bool((got[..., size - 1] == math.inf).all())
    for t in (got, clean[:queries]):
        t[..., [0, 5, size - 1]] = 0
    assert torch.equal(out.view(torch.int16), clean.view(torch.int16))


@pytest.mark.parametrize("spans,prefix", [([(1, 300)] * 3, 0), ([(1, 3000)] * 2, 0), ([(1, 100), (3, 700)], 500), ([(60, 300), (40, 1200)], 0), ([(500, 900), (3, 3)], 40)])
def test_results_in_place_of_the_queries(spans, prefix):
    for heads, kv_heads, size in ((4, 2, 64), (32, 1, 128)):
        b = Batch(spans, prefix, 16, kv_heads, size, seed=2)
        cache, batch = b.on_gpu()
        q = randn(9, b.tokens, heads, size).cuda()
        out = torch.empty_like(q)
        ok(capi.CachedAttention(cache, batch, q, out))
        ok(capi.CachedAttention(cache, batch, q, q))
        assert torch.equal(q.view(torch.int16), out.view(torch.int16))


def test_positions_past_32_bits():
    """Of a length that no page table holds: the entry is not kept, its query turned by its position all the same."""
    b = Batch([(1, 5), (2, 40)], 100, 16, 1, 64)
    b.lengths[0] = (1 << 31) - 1
    cache, batch = b.on_gpu()
    before = b.gpu[0].clone()
    q, k = randn(1, 3, 2, 64), randn(2, 3, 1, 64)
    inv_freq, q_out = capi.rotary_frequencies(64), torch.empty(3, 2, 64, dtype=BF16, device="cuda")
    ok(capi.CacheAppend(cache, batch, k.cuda(), k.cuda(), inv_freq.cuda(), q=q.cuda(), q_out=q_out))
    want, off = oracle.rotated(q, torch.tensor([100 + (1 << 31) - 2, 138, 139]), inv_freq)
    off = off + 2.0 ** 31 * 2.0 ** -51 * (oracle.d(q).abs() + oracle.d(q).abs().roll(32, 2))  # the angle's two roundings in 64 bits, here and in the oracle
    oracle.close(q_out, want, oracle.stored(want, off, BF16), "q")
    changed = (before.view(torch.int16) != b.gpu[0].view(torch.int16)).any(3).any(2).nonzero().tolist()
    assert sorted(changed) == sorted([int(b.table[1, at // 16]), at % 16] for at in (38, 39))


def test_large_logits_and_scales():
    """Logits that grow along the keys, so that the maximum has to be followed, and such that one key has all of the weight."""
    for size, heads, queries in ((64, 4, 1), (128, 4, 40)):
        b = Batch([(queries, 700)], 0, 16, 1, size, values=lambda x: x * 4)
        for scale in (1e-30, 0.01, 1.0, 30.0):
            b.check(heads, scale=scale, what=f"scale {scale}")
        grow = Batch([(queries, 700)], 0, 16, 1, size)
        q = randn(1, grow.tokens, heads, size).abs()
        for i in range(700):  # keys along q
            grow.k[int(grow.table[0, i // 16]), i % 16, 0] = torch.full((size,), 0.02 * i).to(BF16)
        grow.check(heads, scale=0.05, q=q, what="growing")


def test_a_row_with_no_weight_at_all():
    """Keys of -inf logits alone: zeros, and -inf."""
    b = Batch([(1, 20), (1, 3)], 0, 16, 1, 64)
    b.k[int(b.table[1, 0]), :3, 0] = -math.inf
    cache, batch = b.on_gpu()
    q, out, lse = torch.ones(2, 4, 64, dtype=BF16, device="cuda"), torch.full((2, 4, 64), FILL, dtype=BF16, device="cuda"), torch.zeros(2, 4, device="cuda")
    ok(capi.CachedAttention(cache, batch, q, out, lse=lse))
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all()) and bool(torch.isfinite(lse[0]).all())


def test_a_cache_of_more_than_2_to_the_32_bytes():
    """Keys and values at both ends of one, each page's number times its bytes past 32 bits, in slots and in heads outside of them."""
    page, kv_heads, size = 16, 8, 128
    pages = (5 << 30) // (2 * page * kv_heads * size)
    for outer in (False, True):
        whole = torch.empty(pages, *((kv_heads, page) if outer else (page, kv_heads)), size, dtype=BF16, device="cuda")
        view = whole.transpose(1, 2) if outer else whole
        b = Batch([(1, 300), (2, 90)], 40, page, kv_heads, size, seed=11)
        far = torch.randperm(b.pages, generator=torch.Generator().manual_seed(1)) * ((pages - 1) // b.pages)
        far[-1] = pages - 1
        for t in (b.k, b.v):
            t[t.isnan()] = 0
        view[far.cuda()] = b.k.cuda()
        cache = capi.Cache(view, view)
        batch = capi.CacheBatch(b.query_starts.cuda(), b.lengths.cuda(), far[b.table.clamp(0).long()].to(INT32).cuda(), far[b.prefix_pages.long()].to(INT32).cuda(), 40)
        b.v = b.k
        q = randn(2, b.tokens, 16, size)
        out = torch.empty(b.tokens, 16, size, dtype=BF16, device="cuda")
        ok(capi.CachedAttention(cache, batch, q.cuda(), out))
        want, _, bound, _ = b.attention(q, size ** -0.5, True)
        oracle.close(out, want, bound, "far pages")
        k, v = randn(3, b.tokens, kv_heads, size), randn(4, b.tokens, kv_heads, size)
        ok(capi.CacheAppend(cache, batch, k.cuda(), k.cuda()))
        at = int(far[int(b.table[0, 299 // page])])
        assert torch.equal(view[at, 299 % page].cpu(), k[0])
        del whole, view, cache
        torch.cuda.empty_cache()


# ---- appending ----

APPENDS = [  # (queries, length), prefix, page, q heads, kv_heads, size, rotated, first, interleaved
    ([(1, 1)], 0, 16, 4, 1, 64, 64, 0, False), ([(1, 17), (1, 1), (1, 300)], 2048, 16, 32, 8, 128, 128, 0, False), ([(5, 40), (0, 9), (33, 33)], 7, 3, 2, 2, 64, 32, 16, True),
    ([(300, 500), (2, 2)], 0, 64, 6, 3, 96, 48, 0, False), ([(7, 7)], 100, 1, 0, 4, 256, 256, 0, True), ([(9, 20)], 0, 16, 3, 2, 48, 20, 4, False), ([(3, 50)], 0, 16, 4, 2, 32, 0, 0, False),
    ([(2, 30)] * 300, 64, 16, 5, 1, 64, 64, 0, False), ([(1, 1 + 13 * i % 200) for i in range(70)], 5, 16, 8, 2, 128, 64, 64, True),
]


@pytest.mark.parametrize("dtype", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("sequences,prefix,page,heads,kv_heads,size,turned,first,interleaved", APPENDS)
def test_append(sequences, prefix, page, heads, kv_heads, size, turned, first, interleaved, dtype):
    odd = len(sequences) % 2
    b = Batch(sequences, prefix, page, kv_heads, size, dtype, layout=("slots", "heads", "padded")[page % 3], in_front=odd, behind=2)
    tokens = b.tokens
    q, k, v = randn(1, tokens, max(heads, 1), size, scale=3.0), randn(2, tokens, kv_heads, size, scale=3.0), randn(3, tokens, kv_heads, size, scale=3.0)
    inv_freq = capi.rotary_frequencies(turned).cuda() if turned else None
    cache, batch = b.on_gpu()
    before = [x.clone() for x in b.gpu]
    qi, qo = Placed(tokens, max(heads, 1), size, pad=odd, values=q), Placed(tokens, max(heads, 1), size, pad=8, outer=bool(odd))
    ki, vi = Placed(tokens, kv_heads, size, pad=3 * odd, offset=odd, values=k), Placed(tokens, kv_heads, size, outer=True, values=v)
    more = dict(q=qi.view, q_out=qo.view) if heads else {}
    ok(capi.CacheAppend(cache, batch, ki.view, vi.view, inv_freq, interleaved=interleaved, first=first, magnitude=1.5, **more))
    inv_freq = torch.zeros(0) if inv_freq is None else inv_freq.cpu()
    positions = torch.zeros(tokens, dtype=torch.long)
    for i, (n, length) in enumerate(sequences):
        positions[b.starts[i]:b.starts[i] + n] = prefix + length - n + torch.arange(n)
    mine = slice(b.starts[0], b.starts[-1])
    if heads:
        want, off = oracle.rotated(q, positions, inv_freq, interleaved, first, False, 1.5)
        oracle.close(qo.view[mine], want[mine], oracle.stored(want, off, BF16)[mine], "q")
        assert bool((qo.view[:mine.start] == FILL).all()) and bool((qo.view[mine.stop:] == FILL).all()), "queries of padding"
        qo.untouched("q")
    k_want, k_off = oracle.rotated(k, positions, inv_freq, interleaved, first, False, 1.5)
    for got, old, want, off, scales, what in ((b.gpu[0], before[0], k_want, k_off, b.scales[0], "k"), (b.gpu[1], before[1], oracle.d(v), torch.zeros_like(oracle.d(v)), b.scales[1], "v")):
        got = got.cpu()
        kept = torch.ones(got.shape[:2], dtype=torch.bool)
        if scales is not None:  # divided in 32 bits
            want, off = want / scales.double()[:, None], off / scales.double()[:, None] + (want / scales.double()[:, None]).abs() * 2.0 ** -24
            want = want.clamp(-448, 448)
        for i, (n, length) in enumerate(sequences):
            for j in range(n):
                t, at = b.starts[i] + j, length - n + j
                place = int(b.table[i, at // page]), at % page
                kept[place] = False
                oracle.close(got[place], want[t], oracle.stored(want[t], off[t], dtype), f"{what} {i} {j}")
        old, got = ((x.view(torch.uint8) if dtype == E4M3 else x.view(torch.int16)) for x in (old.cpu(), got))
        assert torch.equal(old[kept], got[kept]), f"{what}: written outside of its places"


def test_append_of_tokens_without_a_place():
    """In front of the sequence's entries, past its page table, on pages outside of the cache: nothing is kept of them, their queries are rotated."""
    b = Batch([(5, 3), (2, 40), (3, 60)], 10, 16, 2, 64, spare_columns=0)
    b.lengths[1] = 65  # the last column ends at 64: one of the two is past it
    b.table[2, 3] = -1  # entries 48 .. 63
    cache, batch = b.on_gpu()
    before = b.gpu[0].clone()
    q, k = randn(1, 10, 4, 64), randn(2, 10, 2, 64)
    inv_freq, q_out = capi.rotary_frequencies(64), torch.empty(10, 4, 64, dtype=BF16, device="cuda")
    ok(capi.CacheAppend(cache, batch, k.cuda(), k.cuda(), inv_freq.cuda(), q=q.cuda(), q_out=q_out))
    positions = torch.tensor([10 + 3 - 5 + i for i in range(5)] + [10 + 63, 10 + 64] + [10 + 57 + i for i in range(3)])
    want, off = oracle.rotated(q, positions, inv_freq)
    oracle.close(q_out, want, oracle.stored(want, off, BF16), "q")
    changed = (before.view(torch.int16) != b.gpu[0].view(torch.int16)).any(3).any(2).nonzero().tolist()
    places = [[int(b.table[0, 0]), i] for i in range(3)] + ([[int(b.table[1, 63 // 16]), 63 % 16]] if int(b.table[1, 63 // 16]) >= 0 else [])
    assert sorted(changed) == sorted(places)


def test_append_saturates_and_keeps_what_is_no_number():
    b = Batch([(3, 3)], 0, 16, 1, 32, E4M3)
    cache, batch = b.on_gpu()
    k = torch.zeros(3, 1, 32, dtype=BF16)
    k[0, 0, :4], k[1, 0, 0], k[2, 0, 0] = torch.tensor([1e30, -1e30, math.inf, -math.inf]), math.nan, 1.0
    ok(capi.CacheAppend(cache, batch, k.cuda(), k.cuda()))
    got = b.gpu[1][int(b.table[0, 0]), :3, 0].cpu().float()
    assert got[0, :4].tolist() == [448, -448, 448, -448] and math.isnan(got[1, 0])
    assert float(got[2, 0]) == float((torch.tensor(1.0) / b.scales[1][0]).to(E4M3).float())


def test_quotients_by_any_scale():
    """Values go into an 8-bit cache as x / scale, rounded to 32 bits, then to the type: the same bytes for every scale, from subnormal ones to the largest."""
    scales = torch.tensor([0.013, 1 / 3, 7.7, 2.0 ** -60, 2.0 ** -61 * 1.5, 2.0 ** 60, 2.0 ** 61, 2.0 ** -126, 2.0 ** -140, 1e38, 1.0, 0.0999])
    heads, size, tokens = len(scales), 64, 50
    g = torch.Generator().manual_seed(4)
    v = torch.randn(tokens, heads, size, generator=g) * scales[:, None] * torch.exp2(torch.randint(-12, 11, (tokens, heads, size), generator=g).float())
    v[0, :, :6] = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, 1e38])
    v = v.to(BF16)
    ends = torch.tensor([0, tokens], dtype=INT32).cuda()
    k_cache, v_cache = (torch.zeros(1, tokens, heads, size, dtype=E4M3, device="cuda") for _ in range(2))
    batch = capi.CacheBatch(ends, ends[1:], torch.zeros(1, 1, dtype=INT32).cuda())
    ok(capi.CacheAppend(capi.Cache(k_cache, v_cache, scales.cuda(), scales.cuda()), batch, v.cuda(), v.cuda()))
    want = (v.float() / scales[:, None]).clamp(-448, 448).to(E4M3)
    for got in (k_cache, v_cache):
        got = got[0].cpu()
        same = (got.view(torch.uint8) == want.view(torch.uint8)) | (got.float().isnan() & want.float().isnan())
        assert bool(same.all()), [(float(v[t, h, c]), float(scales[h]), float(got[t, h, c]), float(want[t, h, c])) for t, h, c in (~same).nonzero()[:5].tolist()]


def test_append_with_positions_of_its_own():
    b = Batch([(4, 10), (2, 2)], 0, 16, 2, 64)
    cache, batch = b.on_gpu()
    positions = torch.tensor([7, 3, -9, 100000, 1, 0], dtype=INT32)
    q, inv_freq = randn(1, 6, 2, 64), capi.rotary_frequencies(64)
    there = q.cuda()
    ok(capi.CacheAppend(cache, batch, q.cuda(), q.cuda(), inv_freq.cuda(), q=there, positions=positions.cuda()))  # q in place
    want, off = oracle.rotated(q, positions, inv_freq)
    oracle.close(there, want, oracle.stored(want, off, BF16), "q in place")
    oracle.close(b.gpu[0][int(b.table[0, 0]), 6], want[0], oracle.stored(want, off, BF16)[0], "k")


# ---- together ----

def test_decoding_steps_as_a_user_makes_them():
    """A prompt behind a shared prefix, then token after token: append, attend; lengths go on on the device.  Against attention over all that was ever appended, in 64 bits from
    the unrounded inputs: keys and queries are rounded once (2^-8 of each product's two factors), values and results once."""
    page, heads, kv_heads, size, prefix = 16, 8, 2, 64, 37
    counts = [(20, 5), (1, 1), (70, 3)]
    inv_freq = capi.rotary_frequencies(size)
    b = Batch([(n, n) for n, _ in counts], prefix, page, kv_heads, size, seed=21, spare_columns=3)
    spare = b.pages - 2  # two pages that nobody has yet, in each row's spare columns
    for i in range(3):
        b.table[i, -3:] = -1
    grown = torch.full((b.pages + 12, page, kv_heads, size), math.nan, dtype=BF16)
    caches = []
    for t in (b.k, b.v):
        g = grown.clone()
        g[:b.pages] = t
        caches.append(g.cuda())
    for i in range(3):
        used = -(-counts[i][0] // page)
        for c in range(used, b.table.shape[1]):
            b.table[i, c] = b.pages + 4 * i + c - used if c - used < 4 else -1
    del spare
    lengths = torch.zeros(3, dtype=INT32, device="cuda")
    table, prefix_pages = b.table.cuda(), b.prefix_pages.cuda()
    cache = capi.Cache(*caches)
    history = [([], []) for _ in counts]
    k_prefix, v_prefix = (oracle.placed(t, None, b.prefix_pages.tolist(), page, prefix)[0] for t in (b.k, b.v))
    seed = 100
    for step in range(4):
        new = [n if step == 0 else 1 for n, _ in counts]
        starts = torch.tensor([0, new[0], new[0] + new[1], sum(new)], dtype=INT32)
        lengths += torch.tensor(new, dtype=INT32, device="cuda")
        batch = capi.CacheBatch(starts.cuda(), lengths, table, prefix_pages, prefix)
        tokens = sum(new)
        seed += 1
        qkv = randn(seed, tokens, heads + 2 * kv_heads, size)
        on_gpu = qkv.cuda()
        q, k, v = on_gpu[:, :heads], on_gpu[:, heads:heads + kv_heads], on_gpu[:, heads + kv_heads:]
        out = torch.empty(tokens, heads, size, dtype=BF16, device="cuda")
        ok(capi.CacheAppend(cache, batch, k, v, inv_freq.cuda(), q=q))
        ok(capi.CachedAttention(cache, batch, q, out))
        at = 0
        for i, n in enumerate(new):
            have = len(history[i][0])
            positions = prefix + have + torch.arange(n)
            part = qkv[at:at + n]
            qr, kr = (oracle.rotated(x, positions, inv_freq)[0] for x in (part[:, :heads], part[:, heads:heads + kv_heads]))
            history[i][0].extend(kr)
            history[i][1].extend(part[:, heads + kv_heads:].double())
            keys, values = torch.cat([k_prefix, torch.stack(history[i][0])]), torch.cat([v_prefix, torch.stack(history[i][1])])
            seen = torch.arange(len(keys))[None] <= positions[:, None]
            for h in range(heads):
                want, _, off, _, mass = oracle.attention(qr[:, h], keys[:, h // 4], values[:, h // 4], seen, size ** -0.5)
                worst = size ** -0.5 * (qr[:, h].abs() @ keys[:, h // 4].abs().T).max(1, keepdim=True).values * (2 * 2.0 ** -8 + 2.0 ** -16)
                bound = off + mass * (2 * torch.expm1(worst) + 2.0 ** -8 + 2.0 ** -8) + (want.abs() + mass * 0.1) * 2.0 ** -8
                oracle.close(out[at:at + n, h], want, bound, f"step {step} sequence {i} head {h}")
            at += n


def test_a_block_of_norm_projections_attention_and_transition_runs():
    """The attention half next to the feed-forward half: RMS norm in 8 bits, 8-bit projection, append, attention, 8-bit projection, RMS norm, gated transition; against the same
    steps in 64 bits from what each call was given."""
    import feed_forward_oracle as ff
    tokens, width, heads, kv_heads, size = 6, 512, 8, 2, 64
    b = Batch([(1, 100), (1, 7), (4, 33)], 48, 16, kv_heads, size, seed=31)
    cache, batch = b.on_gpu()
    x, gamma = randn(1, tokens, width).cuda(), (1 + 0.1 * randn(2, width, dtype=FP32)).cuda()
    e8 = lambda *s: torch.empty(*s, dtype=E4M3, device="cuda")
    f32 = lambda *s: torch.empty(*s, device="cuda")
    b16 = lambda *s: torch.empty(*s, dtype=BF16, device="cuda")
    n_qkv = (heads + 2 * kv_heads) * size
    w_qkv, w_o = (randn(3 + i, *s, scale=s[1] ** -0.5).cuda() for i, s in enumerate(((n_qkv, width), (width, heads * size))))
    q8, s8, w8, ws8 = e8(tokens, width), f32(tokens, 4), e8(n_qkv, width), f32(n_qkv // 128, 4)
    qkv = b16(tokens, heads + 2 * kv_heads, size)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    out, o8, os8, wo8, wos8, y, s, n = b16(tokens, heads, size), e8(tokens, heads * size), f32(tokens, 4), e8(width, heads * size), f32(4, 4), b16(tokens, width), b16(tokens, width), b16(tokens, width)
    wg, wu, wd, z = randn(7, 1024, width, scale=width ** -0.5).cuda(), randn(8, 1024, width, scale=width ** -0.5).cuda(), randn(9, width, 1024, scale=1024 ** -0.5).cuda(), b16(tokens, width)
    inv_freq = capi.rotary_frequencies(size).cuda()
    for w, to, scales in ((w_qkv, w8, ws8), (w_o, wo8, wos8)):
        ok(capi.QuantizeFp8(w, to, scales, block_rows=128))
    ok(capi.RmsNorm(x, gamma, out8=q8, scales=s8))
    ok(capi.LinearFp8(q8, s8, w8, ws8, qkv.view(tokens, n_qkv)))
    given = qkv.clone()
    ok(capi.CacheAppend(cache, batch, k, v, inv_freq, q=q))
    b.k, b.v = (t.cpu() for t in b.gpu)
    ok(capi.CachedAttention(cache, batch, q, out))
    ok(capi.QuantizeFp8(out.view(tokens, -1), o8, os8))
    ok(capi.LinearFp8(o8, os8, wo8, wos8, y))
    ok(capi.RmsNorm(y, gamma, residual=x, sum=s, out=n))
    ok(capi.GatedTransition(n, wg, wu, wd, z))
    positions = torch.tensor([48 + 99, 48 + 6] + [48 + 29 + i for i in range(4)])
    want, off = oracle.rotated(given[:, :heads], positions, inv_freq)
    oracle.close(q, want, oracle.stored(want, off, BF16), "rotated q")
    want, _, bound, _ = b.attention(q.cpu(), size ** -0.5, True)
    oracle.close(out, want, bound, "attention")
    assert bool(torch.isfinite(z).all()) and float(z.float().abs().mean()) > 0
    total, norm = ff.rms_norm(y, gamma, 1e-6, x)
    oracle.close(s, total, total.abs() * 2.0 ** -8 * 1.01 + 1e-30, "residual")
    oracle.close(n, norm, norm.abs() * (2.0 ** -8 + ff.norm_slack(width)) * 1.01 + 1e-30, "norm")


def test_captured_and_replayed_with_other_lengths_and_eager_calls_between():
    """A captured step goes on with the lengths, tables and queries that it finds; other streams and calls in between."""
    b = Batch([(1, 900), (1, 3), (1, 200), (1, 64)], 300, 16, 2, 128, seed=41, values=lambda x: x)
    for t in (b.k, b.v):
        t[t.isnan()] = 0.5
    cache, batch = b.on_gpu()
    heads, inv_freq = 8, capi.rotary_frequencies(128).cuda()
    q, k, out, q_out = (torch.empty(4, h, 128, dtype=BF16, device="cuda") for h in (heads, 2, heads, heads))
    rotary = capi.Rotary(q, inv_freq, q_out=q_out)
    append, attend = capi.CacheAppend(cache, batch, k, k, inv_freq, q=q, q_out=q_out), capi.CachedAttention(cache, batch, q_out, out)
    eager_out = torch.empty_like(out)
    eager = capi.CachedAttention(cache, batch, q_out, eager_out)
    lengths = batch.tensors[1]
    q.copy_(randn(1, 4, heads, 128).cuda())
    k.copy_(randn(2, 4, 2, 128).cuda())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for call in (rotary, append, attend):
            assert call.run(side.cuda_stream) == 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for call in (rotary, append, attend):
            assert call.run(side.cuda_stream) == 0
    for i, now in enumerate(([900, 3, 200, 64], [1, 1, 1, 1], [500, 2, 190, 17], [900, 0, 5, 60])):
        lengths.copy_(torch.tensor(now, dtype=INT32, device="cuda"))
        q.copy_(randn(10 + i, 4, heads, 128).cuda())
        out.fill_(FILL)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert eager.run() == 0
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), eager_out.view(torch.int16)), now
        b.k, b.v = (t.cpu() for t in b.gpu)
        b.sequences = [(1, n) for n in now]
        want, _, bound, _ = b.attention(q_out.cpu(), 128 ** -0.5, True)
        oracle.close(out, want, bound, f"{now}")


def test_two_streams_at_once():
    """Calls with workspaces of their own."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for i in range(2):
        b = Batch([(1, 700 + i), (3, 50), (1, 1000)], 200 * i, 16, 2, 64, seed=50 + i)
        q = randn(60 + i, b.tokens, 8, 64)
        cache, batch = b.on_gpu()
        out = torch.empty(b.tokens, 8, 64, dtype=BF16, device="cuda")
        work.append((b, q, out, capi.CachedAttention(cache, batch, q.cuda(), out)))
    torch.cuda.synchronize()
    for _ in range(20):
        for side, (_, _, _, call) in zip(sides, work):
            assert call.run(side.cuda_stream) == 0
    torch.cuda.synchronize()
    for b, q, out, _ in work:
        want, _, bound, _ = b.attention(q, 64 ** -0.5, True)
        oracle.close(out, want, bound, "on a stream of its own")


def test_query_starts_that_fall_stay_in_bounds():
    """Not a call that means anything: nothing outside of the results is written."""
    b = Batch([(3, 30), (4, 40), (2, 20)], 0, 16, 2, 64)
    for starts in ([5, 1, 9, 2], [0, 9, 0, 9], [-100, 1 << 30, -5, 7], [9, 9, 9, 9], [0, 1 << 30, 1 << 30, 1 << 30]):
        b.query_starts = torch.tensor(starts, dtype=INT32)
        cache, batch = b.on_gpu()
        out = Placed(9, 4, 64, pad=8)
        call = capi.CachedAttention(cache, batch, randn(1, 9, 4, 64).cuda(), out.view)
        room = torch.full((call.workspace.numel() + 4096,), 0x55, dtype=torch.uint8, device="cuda")
        at = -room.data_ptr() % 256
        call.args.workspace = room.data_ptr() + at
        ok(call)
        out.untouched(str(starts))
        assert bool((room[at + call.workspace.numel():] == 0x55).all())
        ok(capi.CacheAppend(cache, batch, randn(2, 9, 2, 64).cuda(), randn(3, 9, 2, 64).cuda()))
