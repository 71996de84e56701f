"""The feed-forward operators at the ends of their ranges: hidden layers whose rows are 2^27 bytes apart, values far from one, more rows than one launch has threads."""
import pytest
import torch

import feed_forward_oracle as oracle
from kutacc_amd import capi
from test_gpu_feed_forward import BF16, E4M3, EPS, FP32, Room, cpu_randn, ok, weights_of
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


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows,size", [(3, 7), (5, 64), (9, 300), (4, 2051), (3, 8200)])
def test_rms_norm_of_rows_near_zero_without_eps(dtype, rows, size):
    """Values around 2^-66: 1 / mean(x^2) is past 32 bits, and all results are not."""
    x, dy, gamma = cpu_randn(1, rows, size, scale=2.0 ** -66, dtype=dtype), cpu_randn(2, rows, size, dtype=dtype), 1 + 0.1 * cpu_randn(3, size, dtype=FP32)
    # squares below 2^-126 have steps of 2^-149: the sum of squares is off by size 2^-150 beside some size 2^-132, the factor of a row by half of 2^-18 of itself, and a
    # result by three such factors at most (r, and the r^2 of the pull), beside what the oracle counts
    rows_off = 3 * 2.0 ** -18
    out, dx, dgamma = Room(rows, size, dtype), Room(rows, size, dtype), Room(1, size, FP32)
    ok(capi.RmsNorm(x.cuda(), gamma.cuda(), 0.0, out=out.view))
    _, y = oracle.rms_norm(x, gamma, 0.0)
    oracle.close(out.view, y, oracle.stored(y, y.abs() * (oracle.norm_slack(size) + rows_off), dtype), "out")
    ok(capi.RmsNormBackward(x.cuda(), gamma.cuda(), dy.cuda(), 0.0, grad_x=dx.view, grad_gamma=dgamma.view[0]))
    want, off, want_gamma, off_gamma = oracle.rms_norm_backward(x, gamma, dy, 0.0)
    r = 1 / torch.sqrt((x.double() ** 2).mean(1, keepdim=True))
    h = dy.double() * gamma.double()
    terms = r * (h.abs() + x.double().abs() * r * r * (h * x.double()).abs().mean(1, keepdim=True))
    oracle.close(dx.view, want, oracle.stored(want, off + rows_off * terms, dtype), "grad_x")
    oracle.close(dgamma.view[0], want_gamma, off_gamma + (rows_off + 2.0 ** -24) * (dy.double() * x.double() * r).abs().sum(0), "grad_gamma")


def edges(rows, around):
    """The first and the last rows, and those on either side of `around`."""
    return torch.cat([torch.arange(40), torch.arange(around - 40, around + 40), torch.arange(rows - 40, rows)])


def test_rms_norm_of_more_rows_than_a_launch_has_threads():
    """Eight threads a row: the second of two launches begins behind (2^32 - 1) / 256 workgroups of 32 rows."""
    part = (2 ** 32 - 1) // 256 * 32
    rows, size = part + 1000, 2
    picked = edges(rows, part)
    x, gamma = cpu_randn(1, len(picked), size), 1 + 0.1 * cpu_randn(2, size, dtype=FP32)
    gx, out = torch.zeros(rows, size, device="cuda", dtype=BF16), torch.full((rows, size), 77.0, device="cuda", dtype=BF16)
    gx[picked] = x.cuda()
    out8, scales = torch.full((rows, size), 0x33, device="cuda", dtype=torch.uint8).view(E4M3), torch.full((rows, 1), 77.0, device="cuda")
    ok(capi.RmsNorm(gx, gamma.cuda(), EPS, out=out, out8=out8, scales=scales))
    near = [torch.empty(len(picked), size, device="cuda", dtype=t) for t in (BF16, E4M3)] + [torch.empty(len(picked), 1, device="cuda")]
    ok(capi.RmsNorm(x.cuda(), gamma.cuda(), EPS, out=near[0], out8=near[1], scales=near[2]))
    for got, want in zip((out, out8, scales), near):
        assert torch.equal(got.view(torch.uint8)[picked.cuda()], want.view(torch.uint8))
    _, y = oracle.rms_norm(x, gamma, EPS)
    oracle.close(near[0], y, oracle.stored(y, y.abs() * oracle.norm_slack(size), BF16) + 1e-40, "out")
    assert int(out.count_nonzero()) == int(near[0].count_nonzero()) and int(out8.view(torch.uint8).count_nonzero()) == int(near[1].view(torch.uint8).count_nonzero())
    assert int((scales == 2.0 ** -126).sum()) == rows - len(picked)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantiser_of_more_rows_than_a_launch_has_threads(block_rows):
    """16 threads a row, or two a row of a block of 128."""
    part = (2 ** 32 - 1) // 256 * (16 if block_rows == 1 else 128)
    rows, size = part + 1000, 1
    picked = edges(rows, part)
    x = torch.zeros(rows, size, dtype=BF16, device="cuda")
    x[picked] = cpu_randn(1, len(picked), size).cuda()
    out, scales = torch.full((rows, size), 0x33, device="cuda", dtype=torch.uint8).view(E4M3), torch.full((-(-rows // block_rows), 1), 77.0, device="cuda")
    ok(capi.QuantizeFp8(x, out, scales, block_rows))
    blocks = torch.unique(picked // block_rows)
    for b in blocks.tolist():
        at = slice(b * block_rows, min((b + 1) * block_rows, rows))
        want_q, want_s = oracle.quantise(x[at], block_rows)
        assert torch.equal(scales[b].cpu(), want_s[0]) and torch.equal(out[at].cpu().float(), want_q.float()), b
    assert int((scales == 2.0 ** -126).sum()) == scales.numel() - len(blocks) and int(out.view(torch.uint8).count_nonzero()) == int(x.count_nonzero())


def test_gated_transition_of_more_rows_than_small_tiles_have_threads():
    """134 million rows of eight channels: 2^32 threads in tiles of 32 rows, which would be chosen."""
    rows, c = (1 << 27) + 333, 8
    picked = edges(rows, 1 << 27)
    w, x = weights_of(3, c, c), cpu_randn(1, len(picked), c)
    gx, out = torch.zeros(rows, c, device="cuda", dtype=BF16), torch.full((rows, c), 77.0, device="cuda", dtype=BF16)
    gx[picked] = x.cuda()
    ok(capi.GatedTransition(gx, *(t.cuda() for t in w), out))
    want, off = oracle.gated_transition(x, *w, "silu")["out"]
    oracle.close(out[picked.cuda()], want, oracle.stored(want, off, BF16), "out")
    out[picked.cuda()] = 0
    assert not bool(out.any())


@pytest.mark.parametrize("size", [64, 300, 4100])
def test_rms_norm_of_rows_whose_squares_pass_32_bits(size):
    """As the header has it: zeros, and of the backward pass what came by other ways; the rows beside them as always."""
    x, dy, ds = cpu_randn(1, 5, size), cpu_randn(2, 5, size), cpu_randn(3, 5, size)
    x[2] = (x[2].float() * 2.0 ** 70).to(BF16)
    out, dx = Room(5, size, BF16), Room(5, size, BF16)
    ok(capi.RmsNorm(x.cuda(), None, EPS, out=out.view))
    ok(capi.RmsNormBackward(x.cuda(), None, dy.cuda(), EPS, grad_sum=ds.cuda(), grad_x=dx.view))
    assert not bool(out.view[2].any()) and torch.equal(dx.view[2].cpu(), ds[2])
    others = [0, 1, 3, 4]
    _, y = oracle.rms_norm(x[others], None, EPS)
    oracle.close(out.view[others], y, oracle.stored(y, y.abs() * oracle.norm_slack(size), BF16), "out")
    want, off, _, _ = oracle.rms_norm_backward(x[others], None, dy[others], EPS, ds[others])
    oracle.close(dx.view[others], want, oracle.stored(want, off, BF16), "grad_x")


def test_an_owner_may_go_while_its_call_runs():
    """Its workspace's memory is asked for at once and written on another stream, while the call has not begun."""
    rows, c_o, c_i = 300, 256, 512
    w, x = [t.cuda() for t in weights_of(1, c_o, c_i)], cpu_randn(1, rows, c_o).cuda()
    want, out = torch.empty_like(x), torch.empty_like(x)
    call = capi.GatedTransition(x, *w, want)
    ok(call)
    size = call.workspace.numel()
    del call
    side = torch.cuda.Stream()
    for _ in range(5):
        out.fill_(1)
        torch.cuda.synchronize()
        call = capi.GatedTransition(x, *w, out)
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # some ten milliseconds, by the clock
        assert call.run(side.cuda_stream) == 0
        del call
        others = [torch.full((size,), 255, device="cuda", dtype=torch.uint8) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(bool((o == 255).all()) for o in others)
