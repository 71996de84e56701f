"""A prefix that is read once for the batch, and one that each sequence's tiles walk by themselves: the same borders, layouts, masks and uses for both, each test sure of the form that it runs."""
import pytest
import torch

import cached_attention_oracle as oracle
from cached_attention_routes import prefix_is_shared
from kutacc_amd import capi
from test_gpu_cached_attention import BF16, E4M3, FILL, INT32, SHAPES, Batch, Placed, ok, randn

pytestmark = pytest.mark.gpu


class Routed(Batch):
    """A batch that knows its form, and what that keeps of the weights: 16 bits in tiles of up to 16 rows, of a sequence on average or, where the prefix is shared, of the batch."""

    def shared(self, heads):
        return prefix_is_shared(self.page, self.kv_heads, self.size, len(self.sequences), self.tokens, self.columns, self.prefix, heads)

    def coarse(self, group):
        average = -(-self.tokens * group // min(len(self.sequences), self.tokens))
        return 2.0 ** -16 if average <= 16 and (self.tokens * group <= 16 or not self.shared(group * self.kv_heads)) else 2.0 ** -8


# (queries, length) of each sequence, q heads, kv heads: up to 16 rows in the batch; of a sequence, but not in the batch; more of a sequence, its tiles of many rows
SPANS = [([(1, 50), (0, 9), (1, 1), (1, 300)], 2, 2), ([(1, 300), (3, 41), (0, 7), (4, 4), (1, 700)], 8, 2), ([(16, 30), (9, 100), (1, 1), (30, 250)], 4, 1)]


@pytest.mark.parametrize("dtype", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("size", [64, 128, 256])
@pytest.mark.parametrize("spans", range(3))
@pytest.mark.parametrize("rest", [0, 1, 15, 16, 17, 63, 65, 127])
def test_a_shared_prefix_of_any_length(rest, spans, size, dtype):
    """Lengths around the ends of blocks and tiles, masks, layouts, padding in front and behind, strides and addresses."""
    sequences, heads, kv_heads = SPANS[spans]
    variant = rest % 3 + spans
    page = (16, 48, 6)[variant % 3]
    b = Routed(sequences, 1024 + rest, page, kv_heads, size, dtype, layout=("slots", "heads", "padded")[(variant + rest) % 3], in_front=rest % 2, behind=1 + rest % 3, seed=rest)
    assert b.shared(heads)
    for causal in (True, False):
        b.check(heads, causal, pad=3 * (rest % 2), offset=rest % 2, outer=rest % 4 < 2, what=f"{rest} {spans} {size} {causal}")


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
@pytest.mark.parametrize("prefix", [1, 15, 17, 31, 33, 63, 65, 100, 127, 129])
def test_a_prefix_that_tiles_of_few_rows_walk(prefix, causal):
    """With 16 bits of its weights; keys so few that 8 bits would show."""
    for sequences, heads, kv_heads, size, page in (([(1, 50), (0, 9), (1, 1), (3, 200)], 4, 1, 64, 16), ([(1, 40), (2, 33), (1, 0)], 16, 2, 128, 32), ([(1, 1 + 7 * i) for i in range(9)], 8, 1, 64, 6)):
        b = Routed(sequences, prefix, page, kv_heads, size, seed=prefix, behind=1)
        assert not b.shared(heads) and b.coarse(heads // kv_heads) == 2.0 ** -16
        b.check(heads, causal, what=f"{prefix} {size} {causal}")


@pytest.mark.parametrize("sequences,prefix,page,heads,kv_heads,size", [s for s in SHAPES if s[1]])
def test_weights_of_the_shapes_with_a_prefix(sequences, prefix, page, heads, kv_heads, size):
    """By the form that they take."""
    Routed(sequences, prefix, page, kv_heads, size, behind=2).check(heads, what=f"{sequences[:3]} {prefix}")


def test_missing_pages_of_a_shared_prefix():
    for sequences, heads, kv_heads in SPANS:
        b = Routed(sequences, 1030, 16, kv_heads, 64, seed=3)
        b.prefix_pages[0], b.prefix_pages[7], b.prefix_pages[31], b.prefix_pages[-1] = -1, b.pages, 1 << 30, -(1 << 31)
        b.table[0, 0] = b.pages + 3
        assert b.shared(heads)
        b.check(heads, what="missing pages")
        b.prefix_pages[:] = -1  # all of it
        b.check(heads, what="no page")


@pytest.mark.parametrize("prefix", [1024, 1037])
@pytest.mark.parametrize("size", [64, 128])
def test_results_in_place_behind_a_shared_prefix(size, prefix):
    for sequences, heads, kv_heads in SPANS:
        b = Routed(sequences, prefix, 16, kv_heads, size, seed=2, in_front=1, behind=2)
        assert b.shared(heads)
        cache, batch = b.on_gpu()
        q = randn(9, b.tokens, heads, size).cuda()
        out = q.clone()
        ok(capi.CachedAttention(cache, batch, q, out))  # padding as it is
        ok(capi.CachedAttention(cache, batch, q, q))
        assert torch.equal(q.view(torch.int16), out.view(torch.int16))


def test_what_is_not_seen_behind_a_shared_prefix_may_be_anything():
    for queries, heads in ((3, 4), (30, 2)):
        b = Routed([(queries, queries + 10), (2, 90)], 1000, 16, 1, 64, seed=5)
        assert b.shared(heads)
        q = randn(9, b.tokens, heads, 64).cuda()
        cache, batch = b.on_gpu()
        clean, out = torch.empty_like(q), torch.empty_like(q)
        ok(capi.CachedAttention(cache, batch, q, clean))
        last = queries + 9  # seen by the sequence's last token alone
        place = int(b.table[0, last // 16]), last % 16
        b.gpu[0][place[0], place[1], 0, 3], b.gpu[1][place[0], place[1], 0, 1] = float("nan"), float("inf")
        ok(capi.CachedAttention(cache, batch, q, out))
        rest = [i for i in range(b.tokens) if i != queries - 1]
        assert torch.equal(out[rest].view(torch.int16), clean[rest].view(torch.int16)) and bool(torch.isnan(out[queries - 1]).any(1).all())


def test_a_shared_prefix_past_2_to_the_32_bytes():
    page, kv_heads, size, prefix = 16, 8, 128, 1037
    pages = (5 << 30) // (2 * page * kv_heads * size)
    for outer in (False, True):
        whole = torch.empty(pages, *((kv_heads, page) if outer else (page, kv_heads)), size, dtype=BF16, device="cuda")
        view = whole.transpose(1, 2) if outer else whole
        b = Routed([(1, 300), (2, 90)], prefix, page, kv_heads, size, seed=11)
        assert b.shared(16)
        far = torch.randperm(b.pages, generator=torch.Generator().manual_seed(1)) * ((pages - 1) // b.pages)
        far[-1] = pages - 1
        for t in (b.k, b.v):
            t[t.isnan()] = 0
        view[far.cuda()] = b.k.cuda()
        batch = capi.CacheBatch(b.query_starts.cuda(), b.lengths.cuda(), far[b.table.clamp(0).long()].to(INT32).cuda(), far[b.prefix_pages.long()].to(INT32).cuda(), prefix)
        b.v = b.k
        q, out = randn(2, b.tokens, 16, size), torch.empty(b.tokens, 16, size, dtype=BF16, device="cuda")
        ok(capi.CachedAttention(capi.Cache(view, view), batch, q.cuda(), out))
        want, _, bound, _ = b.attention(q, size ** -0.5, True)
        oracle.close(out, want, bound, "far pages")
        del whole, view
        torch.cuda.empty_cache()


@pytest.mark.parametrize("heads", [2, 8])
def test_a_captured_step_behind_a_shared_prefix(heads):
    """Few rows in the batch, and more: replayed with other lengths, starts and queries, eager calls and synchronizations between."""
    b = Routed([(1, 900), (2, 30), (1, 200), (1, 64)], 1037, 16, 2, 128, seed=41, behind=2)
    assert b.shared(heads)
    for t in (b.k, b.v):
        t[t.isnan()] = 0.5
    cache, batch = b.on_gpu()
    q, out, eager_out = (torch.zeros(b.tokens, heads, 128, dtype=BF16, device="cuda") for _ in range(3))
    lse, eager_lse = (torch.zeros(b.tokens, heads, device="cuda") for _ in range(2))
    captured, eager = capi.CachedAttention(cache, batch, q, out, lse=lse), capi.CachedAttention(cache, batch, q, eager_out, lse=eager_lse)
    side = torch.cuda.Stream()
    assert captured.run(side.cuda_stream) == 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        assert captured.run(side.cuda_stream) == 0
    for i, (tokens, now) in enumerate((([1, 2, 1, 1], [900, 30, 200, 64]), ([1, 1, 1, 1], [1, 1, 1, 1]), ([0, 3, 2, 2], [500, 2, 190, 17]), ([4, 0, 0, 1], [900, 0, 5, 60]))):
        starts = [i % 2]
        for n in tokens:
            starts.append(starts[-1] + n)
        batch.tensors[0].copy_(torch.tensor(starts, dtype=INT32, device="cuda"))
        batch.tensors[1].copy_(torch.tensor(now, dtype=INT32, device="cuda"))
        q.copy_(randn(10 + i, b.tokens, heads, 128).cuda())
        for t in (out, eager_out, lse, eager_lse):
            t.fill_(FILL)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ok(eager)
        assert torch.equal(out.view(torch.int16), eager_out.view(torch.int16)) and torch.equal(lse, eager_lse), i
        b.starts, b.sequences = starts, list(zip(tokens, now))
        want, want_lse, bound, lse_bound = b.attention(q.cpu(), 128 ** -0.5, True)
        mine = slice(starts[0], starts[-1])
        oracle.close(out[mine], want[mine], bound[mine], f"step {i}")
        oracle.close(lse[mine], want_lse[mine], lse_bound[mine], f"lse of step {i}")
        around = [t for t in range(b.tokens) if not starts[0] <= t < starts[-1]]
        assert bool((out[around] == FILL).all()) and bool((lse[around] == FILL).all())


def test_two_streams_with_a_workspace_each():
    """One splits its keys, the other one shares a prefix: neither's pieces end in the other's results."""
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for i, prefix in enumerate((0, 1500)):
        b = Routed([(1, 1700 + i), (3, 50), (1, 1300)], prefix, 16, 2, 64, seed=50 + i)
        q = randn(60 + i, b.tokens, 8, 64)
        cache, batch = b.on_gpu()
        out = torch.empty(b.tokens, 8, 64, dtype=BF16, device="cuda")
        call = capi.CachedAttention(cache, batch, q.cuda(), out)
        assert call.workspace.numel() > 0 and b.shared(8) == (prefix > 0)
        work.append((b, q, out, call))
    torch.cuda.synchronize()
    for _ in range(20):
        for side, (_, _, _, call) in zip(sides, work):
            assert call.run(side.cuda_stream) == 0
    torch.cuda.synchronize()
    for b, q, out, _ in work:
        want, _, bound, _ = b.attention(q, 64 ** -0.5, True)
        oracle.close(out, want, bound, "on a stream of its own")


# Few rows with split keys, many rows with split keys, shared prefixes of few rows, of many, of many in both.  Whatever the starts are, the kernel keeps tokens within the call's, tiles below
# the most that there can be, and pieces within the workspace by comparisons of its own.
@pytest.mark.parametrize("longest,prefix,heads", [(3000, 0, 4), (3000, 0, 32), (20, 900, 1), (20, 900, 4), (20, 900, 16), (700, 900, 4)])
def test_starts_that_fall_with_a_workspace_stay_in_bounds(longest, prefix, heads):
    """Not a call that means anything: nothing outside of the results and the workspace is written."""
    b = Routed([(3, longest), (4, longest - 8), (2, 20)], prefix, 16, 1, 64)
    for starts in ([5, 1, 9, 2], [0, 9, 0, 9], [-100, 1 << 30, -5, 7], [9, 9, 9, 9], [0, 1 << 30, 1 << 30, 1 << 30], [9, 0, 0, 0]):
        b.query_starts = torch.tensor(starts, dtype=INT32)
        cache, batch = b.on_gpu()
        out, lse = Placed(9, heads, 64, pad=8), torch.full((9 * heads + 64,), FILL, device="cuda")
        call = capi.CachedAttention(cache, batch, randn(1, 9, heads, 64).cuda(), out.view, lse=lse[:9 * heads].view(9, heads))
        size = call.workspace.numel()
        assert size > 0 and b.shared(heads) == (prefix > 0)
        room = torch.full((size + 8192,), 0x55, dtype=torch.uint8, device="cuda")
        at = 4096 + -room.data_ptr() % 256
        call.args.workspace = room.data_ptr() + at
        ok(call)
        out.untouched(str(starts))
        assert bool((lse[9 * heads:] == FILL).all())
        assert bool((room[:at] == 0x55).all()) and bool((room[at + size:] == 0x55).all())
