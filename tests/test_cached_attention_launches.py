"""Which kernels rotary positions, the cache in pages and the attention over it take, with what grids and LDS; without a GPU."""
from unittest import mock

import recorded_launches
from kutacc_amd import capi
from recorded_launches import AT

BF16, FP32, E4M3 = capi.K_BF16, capi.K_FP32, capi.K_E4M3
FAR = 1 << 62


def record(calls):
    """With structures inside of the argument structures, as lists of their fields."""
    inside = recorded_launches.CALLS.replace("setattr(args, k, v)", "setattr(args, k, tuple(v) if isinstance(v, list) else v)")
    with mock.patch.object(recorded_launches, "CALLS", inside):
        return recorded_launches.record(calls)


def attention(sequences, tokens, prefix, heads, kv_heads, size, dtype=BF16, page=16, columns=1 << 16):
    scales = AT if dtype == E4M3 else None
    token, per_page = kv_heads * size, page * kv_heads * size
    cache = [1 << 16, page, kv_heads, size, dtype, 0, AT, per_page, token, size, AT, per_page, token, size, scales, scales]
    batch = [sequences, tokens, AT, AT, AT, columns, columns, AT, prefix]
    heads_of = [AT, heads * size, size]
    return "kutacc_hip_cached_attention", "HipCachedAttentionArgs", dict(cache=cache, batch=batch, q_heads=heads, scale=0.125, causal=1, q=heads_of, out=heads_of, lse=AT, workspace=AT,
                                                                        workspace_bytes=FAR)


def rotary(tokens, heads, k_heads, size, dtype=BF16, rotated=None):
    q, k = [AT, heads * size, size], [AT, k_heads * size, size]
    return "kutacc_hip_rotary", "HipRotaryArgs", dict(tokens=tokens, head_size=size, q_heads=heads, k_heads=k_heads, dtype=dtype, positions=AT,
                                                     rotation=[AT, size // 2 * 2 if rotated is None else rotated, 0, 0, 0, 1.0, 0], q=q, q_out=q, k=k, k_out=k)


def test_kernels_are_opted_into_their_lds_once():
    calls = [attention(s, s * n, prefix, 4 * kv, kv, size, dtype) for s in (1, 3, 64, 300) for n in (1, 7, 500) for prefix in (0, 5, 9000) for kv in (1, 8) for size in (16, 64, 128, 256)
             for dtype in (BF16, E4M3)]
    sizes = {}
    for r in record(calls):
        assert r.rc == 0 and r.launches, r
        for kernel, size in r.opted:
            sizes.setdefault(kernel, set()).add(size)
        for k in r.launches:
            assert k.lds <= max(sizes.get(k.kernel, {64 << 10})) <= 160 << 10, k
    assert len(sizes) >= 10 and all(len(s) == 1 for s in sizes.values()), sizes


def test_no_launch_has_2_to_the_32_threads():
    most = (1 << 30) - 1
    calls = [rotary(t, h, k, size, dtype) for t in (1, 1000, 1 << 24, most) for h, k in ((1, 1), (64, 8)) for size in (1, 2, 37, 128, 512) for dtype in (BF16, FP32)]
    calls += [attention(s, t, prefix, h, kv, size, dtype) for s in (1, 1000, 1 << 20) for t in (1, 1 << 16, 1 << 24, most) for prefix in (0, 100) for h, kv in ((1, 1), (8, 2)) for size in (64, 256)
              for dtype in (BF16, E4M3) if t * h < most]
    launched = 0
    for c, r in zip(calls, record(calls)):
        assert r.rc == 0 or (r.rc == capi.EUNSUPPORTED and not r.launches), (c, r)
        launched += r.rc == 0
        for k in r.launches:
            x, y, z = k.grid
            assert 0 < x < 1 << 31 and 0 < y < 1 << 16 and z == 1 and x * y * k.threads < 1 << 32, (c, k)
    assert launched > len(calls) // 2


def test_few_launches():
    """One kernel where nothing is split or shared, else one more that joins the pieces."""
    alone = [attention(8, 8 * 4096, 0, 32, 8, 128), attention(512, 512, 0, 32, 8, 128), attention(8, 8, 0, 32, 8, 128, columns=60)]
    joined = [attention(8, 8, 0, 32, 8, 128), attention(8, 8, 0, 32, 8, 128, columns=100), attention(1, 1, 0, 8, 8, 128), attention(64, 64, 8192, 32, 8, 128), attention(1, 500, 0, 8, 1, 128)]
    for r in record(alone):
        assert len(r.launches) == 1, r
    for r in record(joined):
        assert len(r.launches) == 2 and "combine_kernel" in r.launches[1].kernel, r
