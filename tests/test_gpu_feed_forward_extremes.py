"""The feed-forward operators at the ends of their ranges: hidden layers whose rows are 2^27 bytes apart, values far from one, more rows than one launch has threads."""
import pytest
import torch

import feed_forward_oracle as oracle
from kutacc_amd import capi
from test_gpu_feed_forward import BF16, Room, cpu_randn, ok
from test_gpu_feed_forward_infinities import operands, same

pytestmark = pytest.mark.gpu


def test_gated_transition_of_a_hidden_layer_whose_rows_are_far_apart():
    """32 rows of 69.4 million hidden units, the last of them 2^32 bytes behind the first: down_w picks units at both ends and around a power of two, so that every row's
    result is a sum of few, its own."""
    rows, c_o, c_i = 32, 8, (1 << 32) // (2 * 31) // 8 * 8 + 4096
    picked = [0, 1, (1 << 23) - 1, 1 << 23, c_i // 2, c_i - 8, c_i - 1, c_i - 4096]
    x = cpu_randn(1, rows, c_o)
    w = [cpu_randn(2, len(picked), c_o), cpu_randn(3, len(picked), c_o), cpu_randn(4, c_o, len(picked))]
    gpu = [torch.ones(c_i, c_o, device="cuda", dtype=BF16) for _ in range(2)] + [torch.zeros(c_o, c_i, device="cuda", dtype=BF16)]
    gpu[0][picked], gpu[1][picked], gpu[2][:, picked] = w[0].cuda(), w[1].cuda(), w[2].cuda()
    out = Room(rows, c_o, BF16)
    ok(capi.GatedTransition(x.cuda(), *gpu, out.view))
    want, off = oracle.gated_transition(x, *w, "silu")["out"]
    # (the bound is of the units that are picked: the others are zeros times their values, and add nothing)
    oracle.close(out.view, want, oracle.stored(want, off, BF16), "out")
    out.untouched("out")


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("scale", [1e14, 1e20, 1e30])
@pytest.mark.parametrize("rows,c_o,c_i", [(17, 96, 64), (50, 256, 64), (100, 64, 96), (9001, 128, 96), (300, 256, 512), (70, 77, 130)])
def test_gated_transition_of_gates_far_from_zero(rows, c_o, c_i, scale, activation):
    """Every other unit's gate far above zero, where the activation is its value and the derivative one, the others' far below, where both are zeros.  All else is
    positive, so that results are within the roundings of their operands and their own."""
    x, w, dy = operands(rows, c_o, c_i)
    x, w[1] = (x.float() * scale).to(BF16), (w[1].float() / scale).to(BF16)
    w[0][1::2] *= -1
    want = oracle.gated_transition(x, *w, activation, dy)
    out, grads = Room(rows, c_o, BF16), dict(grad_x=Room(rows, c_o, BF16), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
    gpu = [t.cuda() for t in w]
    ok(capi.GatedTransition(x.cuda(), *gpu, out.view, activation))
    same(out.view, want["out"][0], "out")
    ok(capi.GatedTransitionBackward(x.cuda(), *gpu, dy.cuda(), activation=activation, **{k: r.view for k, r in grads.items()}))
    for name, r in grads.items():
        same(r.view, want[name][0], name)
