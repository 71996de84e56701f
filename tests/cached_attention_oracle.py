"""Rotary positions, a cache in pages and the attention over it in 64 bits on the CPU, and how far 32-bit arithmetic and the roundings to storage may take a result from them.

A rounding is off by at most half a step (bf16 2^-8, fp32 2^-24, e4m3 2^-4 relative to the value, and 2^-10 below its normal numbers).  A sum of n products in 32 bits is
off by at most n 2^-23 times the sum of the products' magnitudes."""
import math

import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24, torch.float8_e4m3fn: 2.0 ** -4}
ADD = 2.0 ** -23
LARGEST = 448.0


def d(t):
    return None if t is None else t.detach().cpu().double()


def close(got, want, bound, what):
    """Everywhere within `bound`; not-a-number and infinities where the oracle has them."""
    got = d(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    same = (got == want) | torch.isnan(want)
    off = torch.where(same, torch.zeros_like(want), (got - want).abs() / (bound + 1e-300))
    assert off.numel() == 0 or off.max() <= 1.0, f"{what}: {float(off.max()):.3g} times the bound at {int(off.argmax())}"


# ---- rotary positions ----

def rotated(x, positions, inv_freq, interleaved=False, first=0, inverse=False, magnitude=1.0):
    """x [tokens, heads, size] with its pairs turned, and how far 32-bit arithmetic may be off: the angle in half turns is rounded once (2^-25 of at most one, times
    pi), sine and cosine are off by at most two units (2^-23), the magnitude's product and the two of the turn round once each."""
    x, f = d(x), d(inv_freq)
    n = 2 * f.numel()
    angle = d(positions)[:, None] * f * (-1.0 if inverse else 1.0)
    c, s = (magnitude * torch.cos(angle))[:, None], (magnitude * torch.sin(angle))[:, None]
    y, off = x.clone(), torch.zeros_like(x)
    one, two = (slice(first, first + n, 2), slice(first + 1, first + n, 2)) if interleaved else (slice(first, first + n // 2), slice(first + n // 2, first + n))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    slack = abs(magnitude) * (math.pi * 2.0 ** -25 + 2.0 ** -23 + 3 * 2.0 ** -24) * (a.abs() + b.abs())
    off[..., one], off[..., two] = slack, slack
    return y, off


def stored(y, off, dtype):
    """The bound of y, off by `off` before it is rounded to `dtype`."""
    return off + (y.abs() + off) * EPS[dtype] + (2.0 ** -10 if dtype == torch.float8_e4m3fn else 0.0)


# ---- attention ----

def placed(cache, scales, pages, page_size, count):
    """Entries 0 .. count - 1 of `pages` as [count, kv_heads, size], and which of them are there."""
    at = torch.arange(count)
    numbers = torch.tensor(pages, dtype=torch.long)[at // page_size] if count else torch.zeros(0, dtype=torch.long)
    there = (numbers >= 0) & (numbers < cache.shape[0])
    rows = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    rows = rows[numbers.clamp(0, cache.shape[0] - 1), at % page_size].contiguous().view(cache.dtype).double()
    return rows * scales.double()[:, None] if scales is not None else rows, there


def attention(q, k, v, seen, scale):
    """q [rows, size], k and v [keys, size], seen [rows, keys], in 64 bits: results, lse, and their bounds before the weights' and the results' own roundings; also the
    sum of the weights times |v|, which the weights' rounding is relative to."""
    logits = scale * (q @ k.T)
    off = torch.where(seen, scale * (q.abs() @ k.abs().T) * k.shape[1] * ADD + logits.abs() * 2.0 ** -21, torch.zeros_like(logits))
    logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
    most = logits.max(1, keepdim=True).values if k.shape[0] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64)
    p = torch.exp(logits - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = p.sum(1, keepdim=True)
    p = torch.where(total == 0, torch.zeros_like(p), p / total)  # what is no number stays none
    vz = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    out = p @ vz
    mass = p @ vz.abs()
    worst = off.max(1, keepdim=True).values if k.shape[0] else torch.zeros_like(most)  # of a logit
    lse = (torch.where(most == -math.inf, torch.zeros_like(most), most) + torch.log(total))[:, 0]
    slack = 2.0 * torch.expm1(worst) + (k.shape[0] + 100) * ADD
    lse_off = (worst + (k.shape[0] + 100) * ADD)[:, 0] + torch.where(torch.isfinite(lse), lse.abs(), torch.zeros_like(lse)) * 2.0 ** -21
    return out, lse, slack * mass, lse_off, mass
