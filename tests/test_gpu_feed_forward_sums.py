"""Sums over many rows, with every row in sight: a bound that grows with the rows, beside sums that grow with their square root, hides a lost block.  Here every block of
32 rows has a channel of its own, shared with a few others, all terms are positive, and the last row weighs as much as all else of its channel."""
import pytest
import torch

import feed_forward_oracle as oracle
from kutacc_amd import capi
from test_gpu_feed_forward import BF16, EPS, FP32, Room, ok
from test_gpu_feed_forward_infinities import SLACK, positive, same

pytestmark = pytest.mark.gpu


def own_channel(t):
    """t [rows, c], but for the channel of the row's block of 32: zero."""
    rows, c = t.shape
    mine = (torch.arange(rows) // 32 % c)[:, None] == torch.arange(c)
    return torch.where(mine, t, torch.zeros_like(t))


def tail_that_counts(rows, c):
    """A power of two for each row, one but for the last row: there the number of rows that share its channel, and more."""
    sharing = 32 * -(-(-(-rows // 32)) // c)
    factor = torch.ones(rows, 1)
    factor[-1] = 2.0 ** max(0, (sharing - 1).bit_length())
    return factor


# on chip with few and many splits, ragged; tiles with the rows split; widths of no whole pieces; up to 64 rows
@pytest.mark.parametrize("rows,c_o,c_i", [(12289, 128, 512), (33001, 128, 288), (70001, 64, 64), (2049, 64, 96), (8191, 64, 320), (20001, 256, 256), (5003, 264, 1024), (2100, 512, 520),
                                          (5088, 124, 130), (2113, 77, 131), (7829, 128, 1030), (33, 96, 64), (64, 64, 64), (17, 32, 96)])
def test_every_row_is_in_the_gradients_of_the_weights(rows, c_o, c_i):
    x, dy = own_channel(positive(1, rows, c_o)), own_channel((positive(2, rows, c_o).float() * tail_that_counts(rows, c_o)).to(BF16))
    w = [positive(3, c_i, c_o), positive(4, c_i, c_o), positive(5, c_o, c_i)]
    want = oracle.gated_transition(x, *w, "silu", dy)
    grads = dict(grad_x=Room(rows, c_o, BF16), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
    ok(capi.GatedTransitionBackward(x.cuda(), *(t.cuda() for t in w), dy.cuda(), **{k: r.view for k, r in grads.items()}))
    for name, r in grads.items():
        same(r.view, want[name][0], name)
        r.untouched(name)
    # what the check can see: without the last row, or a block of 32 in the middle, no gradient would pass
    for lost in (slice(rows - 1, rows), slice(rows // 64 * 32, rows // 64 * 32 + 32)):
        less = oracle.gated_transition(x[lost], *w, "silu", dy[lost])
        for name in ("grad_gate_w", "grad_up_w", "grad_down_w"):
            assert bool((less[name][0] > 2 * SLACK * want[name][0]).any()), (name, lost)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,size", [(147456, 128), (147399, 128), (20001, 512), (50021, 64), (5003, 4096), (3001, 1000), (700, 9000), (1021, 2051)])
def test_every_row_is_in_the_gradient_of_gamma(rows, size, dtype):
    x = positive(1, rows, size).to(dtype)
    dy = own_channel(positive(2, rows, size).to(dtype))
    dgamma = Room(1, size, FP32)
    ok(capi.RmsNormBackward(x.cuda(), None, dy.cuda(), EPS, grad_gamma=dgamma.view[0]))
    _, _, want, _ = oracle.rms_norm_backward(x, None, dy, EPS)
    # a channel's terms are those of `sharing` rows, beside zeros that add nothing: as many additions in 32 bits, and the factors' own errors
    sharing = 32 * -(-(-(-rows // 32)) // size)
    bound = want.abs() * (oracle.norm_slack(size) + (sharing + 8) * 2.0 ** -24)
    oracle.close(dgamma.view[0], want, bound, "grad_gamma")
    r = 1 / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + EPS)
    least = torch.where(dy > 0, dy.double() * x.double() * r, torch.inf).amin(0)
    assert bool((least[want > 0] > 2 * bound[want > 0]).all())  # any row that is lost is seen
