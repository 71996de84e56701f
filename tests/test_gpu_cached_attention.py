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
        # without the logarithm the sums may be of the rounded weights: off by as much once more
        out.buffer.fill_(FILL)
        ok(capi.CachedAttention(cache, batch, qi.view, out.view, scale=scale, causal=causal))
        oracle.close(out.view[mine], want[mine], bound[mine] + want[mine].abs() * self.coarse(heads // self.kv_heads) * (1 + 2.0 ** -7), f"out without lse {what}")
        out.untouched(what)
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
