"""The feed-forward operators in 64 bits on the CPU, and how far 32-bit sums and the roundings to storage may take a result from them.

A rounding is off by at most half a step: EPS[dtype] relative to the value.  A sum of n products in 32 bits is off by at most n 2^-23 times the
sum of the products' magnitudes (half that for additions that round; a matrix instruction may cut instead)."""
import math

import torch

EPS = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ADD = 2.0 ** -23
BLOCK, LARGEST, SMALLEST_SCALE = 128, 448.0, 2.0 ** -126


def d(t):
    return None if t is None else t.detach().cpu().double()


def close(got, want, bound, what):
    """Everywhere within `bound`; not-a-number and infinities where the oracle has them."""
    got = d(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    same = (got == want) | torch.isnan(want)
    off = torch.where(same, torch.zeros_like(want), (got - want).abs())
    worst = (off / (bound + 1e-300)).max() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {float(worst):.3g} times the bound at {int((off / (bound + 1e-300)).argmax())}"


# ---- RMS norm ----

def rms_norm(x, gamma, eps, residual=None):
    s = d(x) + (d(residual) if residual is not None else 0.0)
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    return s, y * d(gamma) if gamma is not None else y


def norm_slack(size):
    """Relative: y's factor 1 / sqrt(mean) is off by half of what the sum of squares is (8 or 16 a thread, then a tree of 10), and 6 roundings."""
    return (16 + 10) / 2 * ADD + 6 * 2.0 ** -24


def rms_norm_backward(x, gamma, dy, eps, grad_sum=None):
    """Gradients, and the bounds of what 32-bit arithmetic takes off them before any rounding to storage."""
    x, dy = d(x), d(dy)
    n = x.shape[1]
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    h = dy * d(gamma) if gamma is not None else dy
    mean = (h * x).mean(1, keepdim=True)
    dx = r * (h - x * (r * r * mean))
    slack = norm_slack(n)
    off = r * (h.abs() * (slack + 4 * 2.0 ** -24) + x.abs() * r * r * ((h * x).abs().mean(1, keepdim=True) * 30 * ADD + mean.abs() * (3 * slack + 6 * 2.0 ** -24)))
    off = off + r * (x.abs() * (r * r * mean).abs() * 2.0 ** -24)
    if grad_sum is not None:
        dx = dx + d(grad_sum)
        off = off + dx.abs() * 2.0 ** -24
    terms = dy * x * r
    return dx, off, terms.sum(0), terms.abs().sum(0) * (slack + (x.shape[0] + 4) * 2.0 ** -24)


# ---- 8 bits ----

def blocks(x, rows):
    """x cut into blocks of rows x 128, zeros past the end: [row blocks, rows, column blocks, 128]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK, 0, -x.shape[0] % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // BLOCK, BLOCK)


def quantise(x, rows):
    """What the quantiser writes for x: both are roundings of single operations, so these are its bits."""
    x = x.detach().cpu().float()
    b = blocks(x, rows)
    scale = (b.abs().amax((1, 3)) / torch.full((), LARGEST)).clamp_min(SMALLEST_SCALE)
    q = (b / scale[:, None, :, None]).reshape(b.shape[0] * rows, -1)[: x.shape[0], : x.shape[1]]
    return q.to(torch.float8_e4m3fn), scale


def spread(scales, rows, columns, per_row):
    return d(scales).repeat_interleave(per_row, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :columns]


def linear_fp8(a, a_scales, w, w_scales, bias=None, dtype=torch.float32):
    """The product and its bound.  A bf16 result may come from the matrix instructions of 8-bit operands, which add 16 neighbouring products at a time
    and cut each at 2^-13 of the largest: 15 cuts in a group of 16, each at most 2^-13 of the largest value of either operand there."""
    x = d(a.cpu().float()) * spread(a_scales, *a.shape, 1)
    y = d(w.cpu().float()) * spread(w_scales, *w.shape, BLOCK)
    out = x @ y.T
    off = (BLOCK + -(-a.shape[1] // BLOCK) + 4) * ADD * (x.abs() @ y.abs().T)
    if dtype == torch.bfloat16:
        def largest(v):
            v = torch.nn.functional.pad(v.abs(), (0, -v.shape[1] % 16))
            return v.view(v.shape[0], -1, 16).amax(2)
        off = off + 15 * 2.0 ** -13 * (largest(x) @ largest(y).T)
    if bias is not None:
        out = out + d(bias)
        off = off + out.abs() * 2.0 ** -24
    return out, off


# ---- gated transition ----

def act(v, name):
    """The activation, its derivative, and bounds of its first and second derivatives."""
    if name == "silu":
        s = torch.sigmoid(v)
        return v * s, s + v * s * (1 - s), 1.2, 0.6
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + th), 0.5 * (1 + th) + 0.5 * v * (1 - th * th) * c * (1 + 3 * 0.044715 * v * v), 1.2, 1.0


SIGMOID = 2.0 ** -19  # relative, of a sigmoid by the hardware's exponential and reciprocal: a unit each, of an argument rounded up to 2^5 times


def gated_transition(x, gate_w, up_w, down_w, activation, grad_out=None):
    """{"out": (value, bound)} and with grad_out the four gradients; bounds without the last rounding to storage."""
    x, wg, wu, wd = d(x), d(gate_w), d(up_w), d(down_w)
    c_o, c_i = x.shape[1], wg.shape[0]
    half = EPS[torch.bfloat16]
    g, u = x @ wg.T, x @ wu.T
    off_g, off_u = c_o * ADD * (x.abs() @ wg.abs().T), c_o * ADD * (x.abs() @ wu.abs().T)
    a, slope, first, second = act(g, activation)
    off_a = first * off_g + SIGMOID * a.abs()
    h = a * u
    off_h = (off_a * u.abs() + a.abs() * off_u + off_a * off_u) + half * h.abs() * (1 + half)
    result = {"out": (h @ wd.T, off_h @ wd.abs().T + c_i * ADD * (h.abs() @ wd.abs().T))}
    if grad_out is not None:
        dy = d(grad_out)
        dh = dy @ wd
        off_dh = c_o * ADD * (dy.abs() @ wd.abs())
        off_slope = second * off_g + SIGMOID * (1 + g.abs())
        dg, du = dh * u * slope, dh * a
        off_dg = (off_dh * u.abs() + dh.abs() * off_u) * (first + off_slope) + (dh * u).abs() * off_slope + half * dg.abs() * (1 + half)
        off_du = off_dh * (a.abs() + off_a) + dh.abs() * off_a + half * du.abs() * (1 + half)
        rows = x.shape[0]
        result["grad_x"] = (dg @ wg + du @ wu, off_dg @ wg.abs() + off_du @ wu.abs() + 2 * c_i * ADD * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()))
        result["grad_gate_w"] = (dg.T @ x, off_dg.T @ x.abs() + rows * ADD * (dg.abs().T @ x.abs()))
        result["grad_up_w"] = (du.T @ x, off_du.T @ x.abs() + rows * ADD * (du.abs().T @ x.abs()))
        result["grad_down_w"] = (dy.T @ h, dy.abs().T @ off_h + rows * ADD * (dy.abs().T @ h.abs()))
    return result


def stored(value, bound, dtype):
    """The bound with the last rounding, to storage."""
    return bound + EPS[dtype] * (value.abs() + bound)
