"""The operators of the attention half of a transformer block, each as a user's program calls it and in plain form.

  op         entry point
  rotary     kutacc_hip_rotary: rotary positions of queries and keys, forward and (`inverse`) for gradients
  append     kutacc_hip_cache_append: new keys, rotated, and values into a paged cache of bf16 or e4m3; new queries rotated in the same pass
  attention  kutacc_hip_cached_attention: attention over a shared prefix and each sequence's own pages, from one token each to whole prompts
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
LARGEST = 448.0  # of e4m3


def listed():
    return [
        # Sixteen sequences decoding one token each: latency is all there is.
        dict(name="rotary_16x40x128", op="rotary", dtype="bf16", tokens=16, heads=32, kv_heads=8, head_size=128, rotated=128, interleaved=False, inverse=False,
             start=5000, factor=1.0),
        # A batch of prompts inside one buffer of queries, keys and values, at positions of a context stretched eight times.
        dict(name="rotary_8191x40x128", op="rotary", dtype="bf16", tokens=8191, heads=32, kv_heads=8, head_size=128, rotated=128, interleaved=False, inverse=False,
             start=120000, factor=8.0),
        # Gradients in fp32: neighbouring channels are pairs, two thirds of a head are rotated.
        dict(name="rotary_backward_fp32_5001x16x96", op="rotary", dtype="fp32", tokens=5001, heads=12, kv_heads=4, head_size=96, rotated=64, interleaved=True,
             inverse=True, start=0, factor=1.0),
        # Decoding: a token each of 32 sequences, behind a shared prefix.
        dict(name="append_32", op="append", cache="bf16", sequences=32, queries_low=1, queries_high=1, shortest=1, longest=1500, prefix=2048, page=16, heads=32,
             kv_heads=8, head_size=128, rotated=128, interleaved=False),
        # Prompts of any length on their way into the cache.
        dict(name="append_prompts", op="append", cache="bf16", sequences=9, queries_low=200, queries_high=1700, shortest=200, longest=2500, prefix=0, page=64, heads=32,
             kv_heads=8, head_size=128, rotated=128, interleaved=False),
        # The same into an 8-bit cache of heads of 64, half of each rotated.
        dict(name="append_fp8_64", op="append", cache="e4m3", sequences=21, queries_low=1, queries_high=300, shortest=300, longest=900, prefix=77, page=16, heads=12,
             kv_heads=12, head_size=64, rotated=32, interleaved=True),
        # The smallest batch that decodes: eight sequences of very different lengths, no prefix.
        dict(name="decode_8", op="attention", cache="bf16", sequences=8, queries_low=1, queries_high=1, shortest=1, longest=1500, prefix=0, page=16, heads=32, kv_heads=8,
             head_size=128, lse=False),
        # A proposal of four tokens each to be verified, heads of 64 with keys of their own, a prefix that ends inside a page.
        dict(name="verify_5x4", op="attention", cache="bf16", sequences=5, queries_low=4, queries_high=4, shortest=30, longest=400, prefix=1000, page=16, heads=16,
             kv_heads=16, head_size=64, lse=True),
        # 64 answers on one long document.
        dict(name="decode_64_prefix_8192", op="attention", cache="bf16", sequences=64, queries_low=1, queries_high=1, shortest=1, longest=1000, prefix=8192, page=64,
             heads=32, kv_heads=8, head_size=128, lse=False),
        # 256 of them, in 8 bits.
        dict(name="decode_256_prefix_16384_fp8", op="attention", cache="e4m3", sequences=256, queries_low=1, queries_high=1, shortest=100, longest=2000, prefix=16384,
             page=32, heads=32, kv_heads=8, head_size=128, lse=False),
        # One token after a very long text.
        dict(name="decode_1_long", op="attention", cache="bf16", sequences=1, queries_low=1, queries_high=1, shortest=131071, longest=131071, prefix=0, page=16, heads=32,
             kv_heads=8, head_size=128, lse=False),
        # The next pieces of three prompts, behind a shared prefix and what they have in the cache: the matrix cores' rate.
        dict(name="prompts_3_prefix_2000", op="attention", cache="bf16", sequences=3, queries_low=900, queries_high=2000, shortest=2000, longest=2600, prefix=2000,
             page=64, heads=32, kv_heads=8, head_size=128, lse=False),
    ]


def _size(rng, low, high):
    """A size between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention"])
    size = rng.choice([32, 64, 64, 128, 128, 128, 256, 16 * rng.randint(2, 16)])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8]) if kv_heads < 16 else 16
    rotated = rng.choice([size, size, size // 2, size // 16 * 8])
    if op == "rotary":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        tokens = _size(rng, 1, max(1, (40 << 20) // ((heads + kv_heads) * size * (2 if dtype == "fp32" else 1))))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=heads, kv_heads=kv_heads, head_size=size, rotated=rotated, interleaved=rng.random() < 0.4,
                    inverse=rng.random() < 0.4, start=rng.choice([0, 0, _size(rng, 1, 1 << 20)]), factor=rng.choice([1.0, 1.0, 4.0, 32.0]))
    case = dict(op=op, cache=rng.choice(["bf16", "bf16", "e4m3"]), prefix=rng.choice([0, _size(rng, 1, 16384), 64 * _size(rng, 1, 128)]), page=rng.choice([1, 16, 16, 32, 64, 128]),
                heads=heads, kv_heads=kv_heads, head_size=size)
    row = kv_heads * size
    if op == "append":
        sequences = _size(rng, 1, 256)
        high = rng.choice([1, _size(rng, 1, max(1, (8 << 20) // ((heads + 2 * kv_heads) * size * sequences)))])
        low = rng.randint(1, high)
        shortest = low + rng.randint(high - low, 500) if high - low < 500 else high
        longest = min(shortest + _size(rng, 1, 2000), max(shortest, (64 << 20) // (row * sequences)))
        case.update(sequences=sequences, queries_low=low, queries_high=high, shortest=max(shortest, high), longest=max(longest, high), rotated=rotated, interleaved=rng.random() < 0.4)
        return case
    kind = rng.choice(["decode", "decode", "verify", "prompts"])
    if kind == "prompts":
        sequences = _size(rng, 1, 8)
        high = _size(rng, 16, max(16, min(4096, (1 << 17) // (sequences * heads))))
        low = rng.randint(1, high)
    else:
        sequences = _size(rng, 1, 256)
        low = high = 1 if kind == "decode" else rng.randint(2, 8)
    shortest = high + rng.choice([0, _size(rng, 1, 1000)])
    longest = shortest + rng.choice([0, _size(rng, 1, 8000)])
    # no more than 400 MB of own keys and values, and no more than 2^37 operations
    longest = max(shortest, min(longest, (100 << 20) // (row * sequences)))
    while 4 * size * heads * sequences * high * (case["prefix"] + longest) > 1 << 37 and case["prefix"] > 1:
        case["prefix"] //= 2
    case.update(sequences=sequences, queries_low=low, queries_high=high, shortest=shortest, longest=longest, lse=rng.random() < 0.3)
    return case


def _ragged(n, low, high):
    """n sizes from low to high, spread evenly and in no order."""
    return [low + int((high - low) * ((i * 0.6180339887498949) % 1.0) + 0.5) for i in range(n)]


def _batch(case):
    """(queries, length) of each sequence."""
    queries = _ragged(case["sequences"], case["queries_low"], case["queries_high"])
    lengths = _ragged(case["sequences"], case["shortest"], case["longest"])
    return [(q, max(q, n)) for q, n in zip(queries, lengths[::-1])]


# ---- inputs ----

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device="cuda", generator=g).to(dtype)

    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    s = dict(case=case)
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["head_size"]
    if "rotated" in case:
        exponents = torch.arange(0, case["rotated"], 2, device="cuda", dtype=torch.float64) / case["rotated"]
        s["inv_freq"] = (10000.0 ** -exponents / case.get("factor", 1.0)).float()
    if case["op"] == "rotary":
        dt, tokens = TYPES[case["dtype"]], case["tokens"]
        qkv = normal(tokens, heads + 2 * kv_heads, size, dtype=dt)  # as one projection leaves them
        s["q"], s["k"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads]
        s["positions"] = case["start"] + torch.randperm(2 * tokens, device="cuda", generator=g, dtype=torch.int32)[:tokens].sort().values
        s["q_out"], s["k_out"] = empty(tokens, heads, size, dtype=dt), empty(tokens, kv_heads, size, dtype=dt)
        if own:
            from kutacc_amd import capi
            s["calls"] = [capi.Rotary(s["q"], s["inv_freq"], s["positions"], k=s["k"], q_out=s["q_out"], k_out=s["k_out"], interleaved=case["interleaved"],
                                      inverse=case["inverse"], magnitude=_magnitude(case))]
        return s

    page, prefix = case["page"], case["prefix"]
    batch = s["batch"] = _batch(case)
    counts = [-(-n // page) for _, n in batch]
    shared = -(-prefix // page)
    pages = shared + sum(counts) + 3
    order = torch.randperm(pages, device="cuda", generator=g, dtype=torch.int32)
    s["prefix_pages"] = order[:shared].clone()
    s["page_table"] = torch.full((len(batch), max(counts)), -1, device="cuda", dtype=torch.int32)
    at = shared
    for i, n in enumerate(counts):
        s["page_table"][i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for q, _ in batch:
        starts.append(starts[-1] + q)
    tokens = starts[-1]
    s["query_starts"] = torch.tensor(starts, device="cuda", dtype=torch.int32)
    s["lengths"] = torch.tensor([n for _, n in batch], device="cuda", dtype=torch.int32)
    s["k_scales"] = s["v_scales"] = None
    if case["cache"] == "e4m3":
        s["k_scales"] = 0.008 + 0.008 * torch.rand(kv_heads, device="cuda", generator=g)
        s["v_scales"] = 0.008 + 0.008 * torch.rand(kv_heads, device="cuda", generator=g)

    def cache(scales):
        x = torch.randn(pages, page, kv_heads, size, device="cuda", generator=g)
        if scales is not None:
            x = (x / scales[:, None]).clamp(-LARGEST, LARGEST)
        return x.to(TYPES[case["cache"]])

    s["k_cache"], s["v_cache"] = cache(s["k_scales"]), cache(s["v_scales"])
    if case["op"] == "append":
        qkv = normal(tokens, heads + 2 * kv_heads, size)
        s["q"], s["k"], s["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        s["q_out"] = empty(tokens, heads, size)
    else:
        s["q"], s["out"] = normal(tokens, heads, size), empty(tokens, heads, size)
        s["lse"] = empty(tokens, heads, dtype=torch.float32) if case["lse"] else None
    if own:
        from kutacc_amd import capi
        c = capi.Cache(s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"])
        b = capi.CacheBatch(s["query_starts"], s["lengths"], s["page_table"], s["prefix_pages"], prefix)
        if case["op"] == "append":
            s["calls"] = [capi.CacheAppend(c, b, s["k"], s["v"], s["inv_freq"], q=s["q"], q_out=s["q_out"], interleaved=case["interleaved"])]
        else:
            s["calls"] = [capi.CachedAttention(c, b, s["q"], s["out"], lse=s["lse"])]
    return s


def _magnitude(case):
    """What goes with a stretched context: its logits grow with the logarithm of the factor."""
    return 0.1 * math.log(case["factor"]) + 1.0


# ---- one pass ----

def run(state):
    op = state["case"]["op"]
    if own:
        for call in state["calls"]:
            rc = call.run()
            if rc != 0:
                raise RuntimeError(f"the library returned {rc}")
        keys = dict(rotary=("q_out", "k_out"), append=("q_out", "k_cache", "v_cache"), attention=("out", "lse"))[op]
        return tuple(state[k] for k in keys)
    return dict(rotary=_rotary, append=_append, attention=_attention)[op](state)


def _rotate(x, positions, inv_freq, interleaved, inverse=False, magnitude=1.0):
    """fp32 of x [tokens, heads, size], the first 2 len(inv_freq) channels of each head rotated."""
    x = x.float()
    n = 2 * inv_freq.numel()
    angles = positions.double()[:, None] * inv_freq.double()
    c, s = (magnitude * torch.cos(angles)).float()[:, None], (magnitude * torch.sin(angles)).float()[:, None]
    if inverse:
        s = -s
    y = x.clone()
    first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def _rotary(s):
    case = s["case"]
    return tuple(_rotate(s[k], s["positions"], s["inv_freq"], case["interleaved"], case["inverse"], _magnitude(case)).to(s[k].dtype) for k in ("q", "k"))


def _places(s):
    """Of each new token its position, page and slot."""
    case = s["case"]
    starts, lengths, page = s["query_starts"].long(), s["lengths"].long(), case["page"]
    tokens = s["q"].shape[0]
    token = torch.arange(tokens, device="cuda")
    sequence = torch.searchsorted(starts, token, right=True) - 1
    at = token - starts[sequence + 1] + lengths[sequence]
    return at + case["prefix"], s["page_table"][sequence, at // page].long(), at % page


def _append(s):
    case = s["case"]
    positions, pages, slots = _places(s)
    k = _rotate(s["k"], positions, s["inv_freq"], case["interleaved"])
    v = s["v"].float()
    if case["cache"] == "e4m3":
        k = (k / s["k_scales"][:, None]).clamp(-LARGEST, LARGEST)
        v = (v / s["v_scales"][:, None]).clamp(-LARGEST, LARGEST)
    for cache, x in ((s["k_cache"], k), (s["v_cache"], v)):
        whole = cache.view(torch.uint8) if case["cache"] == "e4m3" else cache
        x = x.to(cache.dtype)
        whole[pages, slots] = x.view(torch.uint8) if case["cache"] == "e4m3" else x
    q = _rotate(s["q"], positions, s["inv_freq"], case["interleaved"]).to(s["q"].dtype)
    return q, s["k_cache"], s["v_cache"]


def _rows_of_cache(cache, scales, pages, count):
    """fp32 [kv_heads, count, size] of the keys or values on `pages`."""
    raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    x = raw[pages.long()].view(cache.dtype).float().flatten(0, 1)[:count].transpose(0, 1)
    return (x if scales is None else x * scales[:, None, None]).contiguous()


def _attention(s):
    case = s["case"]
    heads, kv_heads, size, prefix, page = (case[k] for k in ("heads", "kv_heads", "head_size", "prefix", "page"))
    tokens, group = s["q"].shape[0], heads // kv_heads
    q = s["q"].float().view(tokens, kv_heads, group, size).transpose(0, 1) * size ** -0.5  # [kv_heads, tokens, group, size]
    q = q.reshape(kv_heads, tokens * group, size)
    out, lse = torch.empty_like(s["out"]), torch.empty(tokens, heads, device="cuda")
    if prefix:  # once for all rows
        pk, pv = (_rows_of_cache(s[c + "_cache"], s[c + "_scales"], s["prefix_pages"], prefix) for c in "kv")
    at = 0
    for i, (n, length) in enumerate(s["batch"]):
        table = s["page_table"][i, :-(-length // page)]
        k, v = (_rows_of_cache(s[c + "_cache"], s[c + "_scales"], table, length) for c in "kv")
        if prefix:
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        logits = q[:, at * group:(at + n) * group] @ k.transpose(1, 2)
        if n > 1:
            query = torch.arange(n, device="cuda").repeat_interleave(group)[:, None]
            logits.masked_fill_(torch.arange(k.shape[1], device="cuda") > query + (k.shape[1] - n), -math.inf)
        most = logits.amax(-1, keepdim=True)
        p = torch.exp(logits.sub_(most))
        total = p.sum(-1, keepdim=True)
        o = (p @ v) / total
        out[at:at + n] = o.view(kv_heads, n, group, size).transpose(0, 1).reshape(n, heads, size).to(out.dtype)
        lse[at:at + n] = (most + torch.log(total)).view(kv_heads, n, group).transpose(0, 1).reshape(n, heads)
        at += n
    return out, lse if case["lse"] else None


# ---- what a pass cannot do without ----

def work(case):
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["head_size"]
    if case["op"] == "rotary":
        n = case["tokens"] * (heads + kv_heads)
        return dict(bytes=2 * n * size * TYPES[case["dtype"]].itemsize + 4 * (case["tokens"] + case["rotated"] // 2), flops=3 * n * case["rotated"])
    batch, e = _batch(case), TYPES[case["cache"]].itemsize
    tokens = sum(q for q, _ in batch)
    tables = 4 * (2 * len(batch) + sum(-(-n // case["page"]) for _, n in batch))
    if case["op"] == "append":
        return dict(bytes=tokens * size * (heads * 4 + 2 * kv_heads * (2 + e)) + 4 * (3 * len(batch) + tokens), flops=3 * tokens * (heads + kv_heads) * case["rotated"])
    keys = case["prefix"] + sum(n for _, n in batch)
    pairs = sum(q * (case["prefix"] + n) - q * (q - 1) // 2 for q, n in batch)  # of a query and a key that it sees
    return dict(bytes=2 * e * kv_heads * size * keys + 4 * tokens * heads * size + 4 * case["lse"] * tokens * heads + tables + 4 * -(-case["prefix"] // case["page"]),
                flops=4 * size * heads * pairs)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    """8-bit results before their rounding: the value over its head's scale."""
    s = prepare(case, seed)

    def turned(x, positions, inverse=False, magnitude=1.0):
        """Pairs as complex numbers, times the unit of their angle."""
        x = x.double()
        n = 2 * s["inv_freq"].numel()
        sign = -1.0 if inverse else 1.0
        angle = sign * torch.outer(positions.double(), s["inv_freq"].double())
        unit = torch.polar(torch.full_like(angle, magnitude), angle).unsqueeze(1)
        part = x[..., :n]
        z = torch.complex(part[..., 0::2].contiguous(), part[..., 1::2].contiguous()) if case["interleaved"] else torch.complex(*(h.contiguous() for h in part.chunk(2, -1)))
        z = z * unit
        part = torch.stack([z.real, z.imag], -1).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
        return torch.cat([part, x[..., n:]], -1)

    if case["op"] == "rotary":
        return tuple(turned(s[k], s["positions"], case["inverse"], _magnitude(case)) for k in ("q", "k"))
    page, prefix = case["page"], case["prefix"]
    if case["op"] == "append":
        k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
        positions = torch.cat([torch.arange(n - q, n) for q, n in s["batch"]]).cuda() + prefix
        k, v = turned(s["k"], positions), s["v"].double()
        if case["cache"] == "e4m3":
            k, v = (x / s[name].double()[None, :, None] for x, name in ((k, "k_scales"), (v, "v_scales")))
            k, v = (torch.minimum(torch.maximum(x, torch.full_like(x, -LARGEST)), torch.full_like(x, LARGEST)) for x in (k, v))
        table = s["page_table"].cpu().tolist()
        flat = torch.tensor([table[i][p // page] * page + p % page for i, (q, n) in enumerate(s["batch"]) for p in range(n - q, n)], device="cuda")
        k_cache.flatten(0, 1)[flat] = k
        v_cache.flatten(0, 1)[flat] = v
        return turned(s["q"], positions), k_cache, v_cache
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["head_size"]
    group = heads // kv_heads
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    order = torch.arange(prefix + case["longest"] + case["queries_high"], device="cuda")
    at = 0
    for i, (n, length) in enumerate(s["batch"]):
        own_pages = s["page_table"][i][order[:length] // page].long()
        pages = torch.cat([s["prefix_pages"][order[:prefix] // page].long(), own_pages])
        slots = torch.cat([order[:prefix] % page, order[:length] % page])
        sees = order[:prefix + length][None, :] <= prefix + length - n + order[:n][:, None]
        for h in range(kv_heads):
            k, v = (_picked(s[c + "_cache"], pages, slots, h) for c in "kv")
            if case["cache"] == "e4m3":
                k, v = k * s["k_scales"][h].double(), v * s["v_scales"][h].double()
            for j in range(h * group, (h + 1) * group):
                logits = torch.mm(s["q"][at:at + n, j].double(), k.T) / math.sqrt(size)
                logits = torch.where(sees, logits, torch.full_like(logits, -math.inf))
                lse[at:at + n, j] = torch.logsumexp(logits, 1)
                out[at:at + n, j] = torch.mm(torch.softmax(logits, 1), v)
        at += n
    return out, lse if case["lse"] else None


def _picked(cache, pages, slots, head):
    raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    return raw[pages, slots, head].view(cache.dtype).double()
