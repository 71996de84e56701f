"""What rotary positions, the cache in pages and the attention over it refuse, before anything is launched, and the frequencies: these run without a GPU."""
import ctypes
import math

import pytest
import torch

from kutacc_amd import capi

AT = 1 << 32  # an address that nothing reads
BF16, E4M3, INT32, FP32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32, torch.float32


def put(struct, fields):
    """Fields by name; those of a structure inside as inside__name."""
    for name, value in fields.items():
        at = struct
        *outer, last = name.split("__")
        for o in outer:
            at = getattr(at, o)
        setattr(at, last, value)


def rotary(**over):
    a = capi.HipRotaryArgs()
    put(a, {**dict(tokens=4, head_size=64, q_heads=8, k_heads=2, dtype=capi.K_BF16, positions=AT, rotation__inv_freq=AT, rotation__rotated=64, rotation__magnitude=1.0), **over})
    for name, heads in (("q", 8), ("q_out", 8), ("k", 2), ("k_out", 2)):
        for field, value in (("data", AT + (64 if name.endswith("out") else 0)), ("token_stride", heads * 64), ("head_stride", 64)):
            if f"{name}__{field}" not in over:
                put(a, {f"{name}__{field}": value})
    return capi.lib().kutacc_hip_rotary(ctypes.byref(a), None)


@pytest.mark.parametrize("over", [
    dict(tokens=-1), dict(tokens=1 << 31), dict(head_size=0), dict(q_heads=0), dict(k_heads=0), dict(q_heads=1 << 31), dict(dtype=0), dict(dtype=capi.K_E4M3),
    dict(rotation__inv_freq=None), dict(rotation__rotated=63), dict(rotation__rotated=66), dict(rotation__rotated=-2), dict(rotation__first=1), dict(rotation__first=-1),
    dict(rotation__rotated=514, head_size=600), dict(rotation__magnitude=math.inf), dict(rotation__magnitude=math.nan), dict(q__data=None, k__data=None), dict(q_out__data=None),
    dict(k_out__data=None), dict(q__token_stride=-1), dict(q__head_stride=-64), dict(q_out__token_stride=8 * 64 - 1), dict(q_out__head_stride=63),
    dict(k_out__token_stride=0), dict(q__token_stride=1 << 40), dict(q_out__data=AT, q__token_stride=1024), dict(q_out__data=AT, q__head_stride=128, q__token_stride=1024),
])
def test_rotary_refuses(over):
    assert rotary(**over) == capi.EINVAL


def test_rotary_of_nothing():
    assert rotary(tokens=0) == 0 and capi.lib().kutacc_hip_rotary(None, None) == capi.EINVAL


SHAPE = dict(cache__pages=10, cache__page_size=16, cache__kv_heads=2, cache__head_size=64, cache__dtype=capi.K_BF16, cache__k=AT, cache__k_page_stride=2048, cache__k_token_stride=128,
             cache__k_head_stride=64, cache__v=AT, cache__v_page_stride=2048, cache__v_token_stride=128, cache__v_head_stride=64, batch__sequences=3, batch__tokens=5,
             batch__query_starts=AT, batch__lengths=AT, batch__page_table=AT, batch__page_table_ld=4, batch__columns=4, batch__prefix_pages=AT, batch__prefix_length=20, q_heads=4)


def append(**over):
    a = capi.HipCacheAppendArgs()
    put(a, {**SHAPE, **dict(rotation__inv_freq=AT, rotation__rotated=64, rotation__magnitude=1.0, q__data=AT, q__token_stride=256, q__head_stride=64, q_out__data=AT + 64,
                            q_out__token_stride=256, q_out__head_stride=64, k__data=AT, k__token_stride=128, k__head_stride=64, v__data=AT, v__token_stride=128, v__head_stride=64), **over})
    return capi.lib().kutacc_hip_cache_append(ctypes.byref(a), None)


def attention(**over):
    a = capi.HipCachedAttentionArgs()
    put(a, {**SHAPE, **dict(scale=0.125, causal=1, q__data=AT, q__token_stride=256, q__head_stride=64, out__data=AT, out__token_stride=256, out__head_stride=64, lse=AT), **over})
    needed = capi.lib().kutacc_hip_cached_attention_workspace(ctypes.byref(a))
    put(a, {**dict(workspace=AT, workspace_bytes=max(needed, 0)), **{k: v for k, v in over.items() if k.startswith("workspace")}})
    return capi.lib().kutacc_hip_cached_attention(ctypes.byref(a), None), needed


BOTH = [
    dict(cache__pages=0), dict(cache__page_size=0), dict(cache__pages=1 << 20, cache__page_size=1 << 11), dict(cache__kv_heads=0), dict(cache__head_size=0), dict(cache__dtype=0),
    dict(cache__dtype=capi.K_FP32), dict(cache__k=None), dict(cache__v=None), dict(cache__k_page_stride=2047), dict(cache__k_token_stride=64), dict(cache__k_head_stride=56),
    dict(cache__v_page_stride=0), dict(cache__v_token_stride=-128), dict(cache__v_head_stride=1 << 40), dict(cache__k_scales=AT), dict(cache__v_scales=AT),
    dict(cache__dtype=capi.K_E4M3), dict(cache__dtype=capi.K_E4M3, cache__k_scales=AT), dict(batch__sequences=-1), dict(batch__tokens=-1), dict(batch__tokens=1 << 31),
    dict(batch__query_starts=None), dict(batch__lengths=None), dict(batch__page_table=None), dict(batch__page_table_ld=3), dict(batch__columns=-1), dict(batch__columns=1 << 28),
    dict(batch__prefix_pages=None), dict(batch__prefix_length=-1), dict(batch__prefix_length=1 << 30),
]
NO_KERNEL = [
    dict(cache__head_size=60, cache__k_head_stride=64), dict(cache__k=AT + 8), dict(cache__v=AT + 2), dict(cache__k_page_stride=2052), dict(cache__v_token_stride=132, cache__v_page_stride=4096),
    dict(cache__dtype=capi.K_E4M3, cache__k_scales=AT, cache__v_scales=AT, cache__k_head_stride=72, cache__k_token_stride=144, cache__k_page_stride=16 * 144),
]


@pytest.mark.parametrize("over", BOTH + [
    dict(rotation__inv_freq=None), dict(rotation__rotated=65), dict(rotation__first=2), dict(q_heads=0), dict(q_out__data=None), dict(q_out__token_stride=255), dict(k__data=None),
    dict(v__data=None), dict(k__token_stride=-1), dict(q_out__data=AT, q__token_stride=512)])
def test_append_refuses(over):
    assert append(**over) == capi.EINVAL


@pytest.mark.parametrize("over", BOTH + [
    dict(q_heads=0), dict(q_heads=3), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(causal=2), dict(q__data=None), dict(out__data=None),
    dict(out__token_stride=255), dict(out__head_stride=0), dict(q__head_stride=-1), dict(workspace=None, batch__prefix_length=1000),
    dict(workspace=AT + 128, batch__prefix_length=1000), dict(workspace_bytes=256, batch__prefix_length=1000)])  # a prefix that is shared: results meet there
def test_attention_refuses(over):
    assert attention(**over)[0] == capi.EINVAL


@pytest.mark.parametrize("over", NO_KERNEL)
def test_what_there_is_no_kernel_for(over):
    rotation = dict(rotation__rotated=0)
    assert append(**over, **rotation) == attention(**over)[0] == capi.EUNSUPPORTED


def test_heads_beyond_the_widest():
    wide = dict(cache__head_size=264, cache__k_head_stride=264, cache__k_token_stride=528, cache__k_page_stride=16 * 528, cache__v_head_stride=264, cache__v_token_stride=528,
                cache__v_page_stride=16 * 528, q__head_stride=264, q__token_stride=4 * 264)
    assert attention(**wide, out__head_stride=264, out__token_stride=4 * 264) == (capi.EUNSUPPORTED, 0)
    assert append(**wide, q_out__head_stride=264, q_out__token_stride=4 * 264, k__head_stride=264, k__token_stride=528, v__head_stride=264, v__token_stride=528) == capi.EUNSUPPORTED


def test_results_in_place_have_the_queries_strides():
    same = dict(q__data=AT, out__data=AT)
    assert attention(**same, out__token_stride=2048)[0] == capi.EINVAL
    assert attention(**same, q__head_stride=128)[0] == capi.EINVAL


def test_calls_that_do_nothing():
    assert append(batch__tokens=0) == append(batch__sequences=0) == 0
    assert attention(batch__tokens=0) == attention(batch__sequences=0) == (0, 0)
    L = capi.lib()
    assert L.kutacc_hip_cache_append(None, None) == L.kutacc_hip_cached_attention(None, None) == L.kutacc_hip_cached_attention_workspace(None) == capi.EINVAL
    assert attention(cache__page_size=0)[1] == attention(q_heads=3)[1] == capi.EINVAL


# ---- frequencies ----

def test_frequencies():
    n, base = 64, 10000.0
    j = torch.arange(n // 2, dtype=torch.float64)
    plain = base ** (-2 * j / n)

    def same(got, want):
        assert got.dtype == FP32 and torch.allclose(got.double(), want, rtol=2.0 ** -23, atol=0)

    same(capi.rotary_frequencies(n), plain)
    same(capi.rotary_frequencies(n, scaling="linear", factor=8.0), plain / 8)
    stretched = capi.rotary_frequencies(n, scaling="base", factor=4.0)
    same(stretched, (base * 4.0 ** (n / (n - 2))) ** (-2 * j / n))
    assert stretched[0] == 1.0 and abs(float(stretched[-1]) / float(plain[-1]) - 0.25) < 1e-6
    length, fast, slow, factor = 4096.0, 32.0, 1.0, 16.0
    turns = length * plain / (2 * math.pi)
    keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
    same(capi.rotary_frequencies(n, scaling="by_turns", factor=factor, original_length=length, fast=fast, slow=slow), plain * keep + plain / factor * (1 - keep))
    pair = lambda t: n * math.log(length / (t * 2 * math.pi)) / (2 * math.log(base))  # turns t times
    low, high = math.floor(pair(fast)), math.ceil(pair(slow))
    mix = ((j - low) / (high - low)).clamp(0, 1)
    got = capi.rotary_frequencies(n, scaling="by_pairs", factor=factor, original_length=length, fast=fast, slow=slow)
    same(got, plain / factor * mix + plain * (1 - mix))
    assert torch.equal(got[:low + 1].double(), plain[:low + 1].float().double()) and bool((got[turns < slow].double() <= plain[turns < slow] / factor * 1.0000002).all())
    same(capi.rotary_frequencies(2), torch.ones(1, dtype=torch.float64))


@pytest.mark.parametrize("args", [(0,), (3,), (514,), (64, 1.0), (64, math.inf), (64, 1e4, "linear", 0.5), (64, 1e4, "linear", math.nan), (2, 1e4, "base", 2.0), (64, 1e4, "by_pairs", 2.0),
                                  (64, 1e4, "by_turns", 2.0, 4096.0, 1.0, 1.0), (64, 1e4, "by_turns", 2.0, 4096.0, 1.0, 0.0), (64, 1e4, "by_pairs", 2.0, -1.0)])
def test_frequencies_refuse(args):
    with pytest.raises(ValueError):
        capi.rotary_frequencies(*args)
    assert capi.lib().kutacc_hip_rotary_frequencies(None, 64, 0, 1e4, 1.0, 0.0, 0.0, 0.0) == capi.EINVAL
    assert capi.lib().kutacc_hip_rotary_frequencies(AT, 64, 5, 1e4, 1.0, 0.0, 0.0, 0.0) == capi.EINVAL


# ---- the Python owners ----

def e(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype)


def parts(**over):
    t = dict(k_cache=e(10, 16, 2, 64), v_cache=e(10, 16, 2, 64), k_scales=None, v_scales=None, query_starts=e(4, dtype=INT32), lengths=e(3, dtype=INT32), page_table=e(3, 4, dtype=INT32),
             prefix_pages=e(2, dtype=INT32), prefix_length=20)
    t.update(over)
    return t


def pair(**over):
    t = parts(**over)
    return (capi.Cache(t["k_cache"], t["v_cache"], t["k_scales"], t["v_scales"]),
            capi.CacheBatch(t["query_starts"], t["lengths"], t["page_table"], t["prefix_pages"], t["prefix_length"]))


def test_cache_owners_refuse_wrong_tensors():
    cache, batch = pair()
    capi.CachedAttention(cache, batch, e(5, 4, 64), e(5, 4, 64), lse=e(5, 4, dtype=FP32))
    capi.CacheAppend(cache, batch, e(5, 2, 64), e(5, 2, 64), e(32, dtype=FP32), q=e(5, 4, 64))
    for over in (dict(v_cache=e(10, 16, 2, 63)), dict(v_cache=e(10, 16, 2, 64, dtype=E4M3)), dict(k_cache=e(10, 16, 2, 64, dtype=FP32)), dict(k_cache=e(10, 16, 64, 2).transpose(2, 3)),
                 dict(k_scales=e(3, dtype=FP32)), dict(query_starts=e(3, dtype=INT32)), dict(lengths=e(3, dtype=torch.int64)), dict(page_table=e(2, 4, dtype=INT32)),
                 dict(page_table=e(4, 3, dtype=INT32).t()), dict(prefix_pages=None), dict(prefix_pages=e(4, dtype=INT32)[::2])):
        with pytest.raises(ValueError):
            pair(**over)
    with pytest.raises(ValueError, match="for a prefix"):
        capi.CachedAttention(*pair(prefix_pages=e(1, dtype=INT32)), e(5, 4, 64), e(5, 4, 64))
    for q, out, more in ((e(5, 4, 64, dtype=FP32), e(5, 4, 64), {}), (e(5, 4, 64), e(5, 4, 65), {}), (e(5, 4, 64), e(4, 4, 64), {}), (e(5, 3, 64), e(5, 3, 64), {}),
                         (e(5, 4, 64), e(5, 4, 64), dict(lse=e(5, 4))), (e(5, 64, 4).transpose(1, 2), e(5, 4, 64), {}), (e(5, 4, 64), e(5, 4, 64).to("meta"), {})):
        with pytest.raises(ValueError):
            capi.CachedAttention(cache, batch, q, out, **more)
    for k, v, more in ((e(5, 3, 64), e(5, 2, 64), {}), (e(5, 2, 64), e(4, 2, 64), {}), (e(5, 2, 64), e(5, 2, 64), dict(q_out=e(5, 4, 64))), (e(5, 2, 64), e(5, 2, 64), dict(inv_freq=e(32))),
                       (e(5, 2, 64), e(5, 2, 64), dict(q=e(5, 4, 64), q_out=e(5, 5, 64))), (e(5, 2, 64), e(5, 2, 64), dict(positions=e(5, dtype=torch.int64)))):
        with pytest.raises(ValueError):
            capi.CacheAppend(cache, batch, k, v, **more)


def test_rotary_owner_refuses_wrong_tensors():
    q, f = e(5, 4, 64), e(32, dtype=FP32)
    capi.Rotary(q, f, e(5, dtype=INT32), k=e(5, 2, 64))
    for bad in (dict(positions=e(4, dtype=INT32)), dict(positions=e(5, dtype=torch.int64)), dict(k=e(5, 2, 32)), dict(k=e(5, 2, 64, dtype=FP32)), dict(q_out=e(5, 3, 64)), dict(k_out=e(5, 2, 64))):
        with pytest.raises(ValueError):
            capi.Rotary(q, f, **bad)
    for q2, f2 in ((q.half(), f), (q, f.double()), (q, e(32, 1, dtype=FP32)), (e(5, 64, 4).transpose(1, 2), f)):
        with pytest.raises(ValueError):
            capi.Rotary(q2, f2)


def test_owners_of_host_tensors_do_not_run(monkeypatch):
    cache, batch = pair()
    calls = [capi.Rotary(e(5, 4, 64), e(32, dtype=FP32)), capi.CacheAppend(cache, batch, e(5, 2, 64), e(5, 2, 64)), capi.CachedAttention(cache, batch, e(5, 4, 64), e(5, 4, 64))]
    monkeypatch.setattr(capi, "lib", lambda: pytest.fail("the library was called"))
    for call in calls:
        with pytest.raises(ValueError, match="not the current GPU"):
            call.run()
