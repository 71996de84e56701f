"""What the rounding of the hidden layer and of its gradients leaves, where calls keep it: results whose terms nearly cancel, so that the rests are most of them."""
import pytest
import torch

import feed_forward_oracle as oracle
from kutacc_amd import capi
from test_gpu_feed_forward import BF16, Room, cpu_randn, ok

pytestmark = pytest.mark.gpu


def nearly(t, seed, by=2.0 ** -5):
    return (t.float() * (1 + by * torch.randn(t.shape, generator=torch.Generator().manual_seed(seed)))).to(BF16)


def cancelling(rows, c_o, c_i):
    """Rows in pairs whose gradients of out are opposite, and units in pairs whose columns of down_w nearly are: what either contributes is the difference."""
    x, dy = cpu_randn(1, rows, c_o), cpu_randn(2, rows, c_o)
    half = rows // 2
    if half:
        x[-half:], dy[-half:] = nearly(x[:half], 3), -dy[:half]
    wg, wu, wd = cpu_randn(4, c_i, c_o, scale=c_o ** -0.5), cpu_randn(5, c_i, c_o, scale=c_o ** -0.5), cpu_randn(6, c_o, c_i, scale=c_i ** -0.5)
    half = c_i // 2
    wg[half:], wu[half:], wd[:, half:] = wg[:half], wu[:half], -nearly(wd[:, :half], 7)
    return x, [wg, wu, wd], dy


def bounds(x, w, activation, dy, monkeypatch):
    """The oracle's, but for operands that are a rounding within 2^-8 and a rest within 2^-8 of that."""
    with monkeypatch.context() as m:
        m.setitem(oracle.EPS, BF16, 2.0 ** -16)
        found = oracle.gated_transition(x, *w, activation, dy)
    return {k: (v, oracle.stored(v, off, BF16)) for k, (v, off) in found.items()}


def with_operands(x, w, activation, dy, kept):
    """The gradients from operands as `kept` holds them, in 64 bits, rounded once."""
    x, dy, wg, wu, wd = (t.double() for t in (x, dy, *w))
    g, u, dh = x @ wg.T, x @ wu.T, dy @ wd
    a, slope, _, _ = oracle.act(g, activation)
    h, dg, du = kept(a * u), kept(dh * u * slope), kept(dh * a)
    return {k: v.to(BF16).double() for k, v in dict(grad_x=dg @ wg + du @ wu, grad_gate_w=dg.T @ x, grad_up_w=du.T @ x, grad_down_w=dy.T @ h).items()}


def rounded(v):
    return v.to(BF16).double()


WRONG = {"no rests": rounded, "rests of the other sign": lambda v: rounded(v) - rounded(v - rounded(v)), "rests of other units": lambda v: rounded(v) + rounded(v - rounded(v)).roll(1, 1)}


# up to 32 rows all four gradients, up to 64 that of x: full and ragged blocks of rows, one block of units and several, fewer channels than waves share and more
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,c_o,c_i", [(1, 32, 32), (2, 64, 96), (5, 32, 64), (17, 96, 64), (32, 32, 96), (31, 288, 32), (33, 32, 64), (50, 96, 32), (64, 64, 96), (40, 288, 32)])
def test_gradients_of_few_rows_keep_what_rounding_leaves(rows, c_o, c_i, activation, monkeypatch):
    x, w, dy = cancelling(rows, c_o, c_i)
    want = bounds(x, w, activation, dy, monkeypatch)
    names = ["grad_x"] + (["grad_gate_w", "grad_up_w", "grad_down_w"] if rows <= 32 else [])
    for how, kept in WRONG.items():  # what the check can see
        for name, got in with_operands(x, w, activation, dy, kept).items():
            value, bound = want[name]
            assert name not in names or bool(((got - value).abs() > bound).any()), (name, how)
    grads = dict(grad_x=Room(rows, c_o, BF16), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
    ok(capi.GatedTransitionBackward(x.cuda(), *(t.cuda() for t in w), dy.cuda(), activation=activation, **{k: r.view for k, r in grads.items()}))
    for name in names:
        oracle.close(grads[name].view, *want[name], name)


# forward: up to 64 rows and 4096 results
@pytest.mark.parametrize("rows,c_o,c_i", [(1, 32, 64), (3, 128, 96), (16, 64, 32), (17, 96, 64), (64, 64, 128)])
def test_few_results_keep_what_rounding_leaves(rows, c_o, c_i, monkeypatch):
    x, w, dy = cancelling(rows, c_o, c_i)
    half = c_i // 2  # here the pairs' hidden values nearly are the same, and their columns opposite
    w = [torch.cat([w[0][:half], nearly(w[0][:half], 8)]), w[1], torch.cat([w[2][:, :half], -w[2][:, :half]], 1)]
    value, bound = bounds(x, w, "silu", dy, monkeypatch)["out"]
    g, u = x.double() @ w[0].double().T, x.double() @ w[1].double().T
    for how, kept in WRONG.items():
        got = rounded(kept(oracle.act(g, "silu")[0] * u) @ w[2].double().T)
        assert bool(((got - value).abs() > bound).any()), how
    out = Room(rows, c_o, BF16)
    ok(capi.GatedTransition(x.cuda(), *(t.cuda() for t in w), out.view))
    oracle.close(out.view, value, bound, "out")
