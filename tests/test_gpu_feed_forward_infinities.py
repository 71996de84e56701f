"""Infinities among the operands of the gated transition and its backward pass: where the definition in 64 bits has an infinity or no number, so has the result, in
every kernel.  All operands are positive, so that sums that meet an infinity are infinities, and finite ones keep their relative accuracy."""
import math

import pytest
import torch

import feed_forward_oracle as oracle
from kutacc_amd import capi
from test_gpu_feed_forward import BF16, Room, ok

pytestmark = pytest.mark.gpu

# Of positive terms, relative: an operand's rounding and the result's, each within 2^-8, and 32-bit sums, the sigmoid and the derivative, below 2^-11 here
# (2048 products at 2^-23 each are 2^-12; the sigmoid's 2^-19 times values of a few)
SLACK = 2 * 2.0 ** -8 * (1 + 2.0 ** -8) + 2.0 ** -11

# few results; up to 16, 32 and 64 rows of the backward pass; on chip, with rows that fill no block of 32; tiles; widths of no whole pieces
SHAPES = [(1, 64, 128), (16, 128, 512), (17, 96, 64), (33, 64, 96), (50, 256, 64), (65, 64, 64), (100, 64, 96), (9001, 128, 96), (300, 256, 512), (70, 77, 130)]


def positive(seed, *shape, scale=1.0):
    return ((0.5 + torch.rand(*shape, generator=torch.Generator().manual_seed(seed))) * scale).to(BF16)


def operands(rows, c_o, c_i):
    x, dy = positive(1, rows, c_o), positive(2, rows, c_o)
    return x, [positive(3, c_i, c_o, scale=1 / c_o), positive(4, c_i, c_o, scale=1 / c_o), positive(5, c_o, c_i, scale=1 / c_i)], dy


PAST_BF16 = (2 - 2.0 ** -8) * 2.0 ** 127  # what rounds to an infinity: the largest value and half a step


def same(got, want, what):
    got = got.cpu().double()
    want = torch.where(want.abs() >= PAST_BF16, want.sign() * math.inf, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: {int(torch.isnan(got).sum())} are no numbers, and should {int(torch.isnan(want).sum())}"
    assert torch.equal(torch.isinf(got), torch.isinf(want)), f"{what}: {int(torch.isinf(got).sum())} infinities, and should be {int(torch.isinf(want).sum())}"
    finite = torch.isfinite(want)
    assert bool((got[finite] - want[finite]).abs().le(SLACK * want[finite].abs()).all()), what


def put_infinity(place, w, dy):
    t = dict(gate_w=w[0], up_w=w[1], down_w=w[2], grad_out=dy)[place]
    t[t.shape[0] // 2, t.shape[1] // 3] = math.inf


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("place", ["gate_w", "up_w", "down_w"])
@pytest.mark.parametrize("rows,c_o,c_i", SHAPES)
def test_gated_transition_keeps_infinities(rows, c_o, c_i, place, activation):
    x, w, dy = operands(rows, c_o, c_i)
    put_infinity(place, w, dy)
    want = oracle.gated_transition(x, *w, activation)["out"][0]
    assert bool(torch.isinf(want).any())
    out = Room(rows, c_o, BF16)
    ok(capi.GatedTransition(x.cuda(), *(t.cuda() for t in w), out.view, activation))
    same(out.view, want, "out")


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("place", ["gate_w", "up_w", "down_w", "grad_out"])
@pytest.mark.parametrize("rows,c_o,c_i", SHAPES + [(12289, 128, 160), (20479, 64, 64)])
def test_gated_transition_backward_keeps_infinities(rows, c_o, c_i, place, activation):
    x, w, dy = operands(rows, c_o, c_i)
    put_infinity(place, w, dy)
    want = oracle.gated_transition(x, *w, activation, dy)
    grads = dict(grad_x=Room(rows, c_o, BF16), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
    ok(capi.GatedTransitionBackward(x.cuda(), *(t.cuda() for t in w), dy.cuda(), activation=activation, **{k: r.view for k, r in grads.items()}))
    for name, r in grads.items():
        same(r.view, want[name][0], name)
