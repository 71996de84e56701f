"""RMS norm, 8-bit linear, gated transition and their backward passes on the GPU, against their definitions in 64 bits."""
import math

import pytest
import torch

import feed_forward_oracle as oracle
from kutacc_amd import capi

pytestmark = pytest.mark.gpu

BF16, FP32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "fp32": FP32}
EPS = 1e-6
FILL = 77.0  # what surrounds a result and has to stay


def cpu_randn(seed, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def placed(t, ld=None, offset=0):
    """t on the GPU with rows `ld` apart, `offset` elements behind an aligned address."""
    rows, size = t.shape
    ld = ld or size
    buffer = torch.full((offset + rows * ld,), FILL, device="cuda", dtype=FP32).to(t.dtype)
    view = buffer[offset:offset + rows * ld].view(rows, ld)[:, :size]
    view.copy_(t.cuda())
    return view


class Room:
    """A result's rows in the middle of a buffer that has to keep what is around them."""

    def __init__(self, rows, size, dtype, ld=None, offset=0, after=3):
        self.rows, self.size, self.ld = rows, size, ld or size
        self.buffer = torch.full((offset + (rows + after) * self.ld,), FILL, device="cuda", dtype=FP32).to(dtype)
        self.all = self.buffer[offset:].view(rows + after, self.ld)
        self.view, self.offset = self.all[:rows, :size], offset

    def untouched(self, what):
        b = self.buffer.float().clone()
        rest = b[self.offset:].view(-1, self.ld)
        rest[:self.rows, :self.size] = FILL_OF[self.buffer.dtype]
        assert bool((b == FILL_OF[self.buffer.dtype]).all()), f"{what}: written outside of its rows"


FILL_OF = {t: float(torch.tensor(FILL).to(t).float()) for t in (BF16, FP32, E4M3)}


def ok(call):
    rc = call.run()
    torch.cuda.synchronize()
    assert rc == 0, rc


# ---- RMS norm ----

SIZES = [1, 7, 8, 63, 64, 65, 128, 130, 256, 257, 512, 1000, 1024, 1030, 2048, 2051, 4096, 4100, 8192, 8200, 16384]


def check_norm(case, x, residual, gamma, sum_, out, out8, scales):
    s, y = oracle.rms_norm(x, gamma, EPS, residual)
    dt = x.dtype
    slack = oracle.norm_slack(x.shape[1])
    if sum_ is not None:
        oracle.close(sum_, s, s.abs() * (oracle.EPS[dt] + 2.0 ** -24), f"{case} sum")
    near = y.abs() * slack
    if out is not None:
        oracle.close(out, y, oracle.stored(y, near, dt) + 1e-40, f"{case} out")
    if out8 is not None:
        amax = oracle.blocks(y, 1).abs().amax((1, 3))
        want = (amax / 448.0).clamp_min(oracle.SMALLEST_SCALE)
        oracle.close(scales, want, want * (slack + 2.0 ** -23), f"{case} scales")
        held = out8.cpu().float().double() * oracle.spread(scales, *y.shape, 1)
        step = torch.maximum(y.abs() * 2.0 ** -4, oracle.spread(scales, *y.shape, 1) * 2.0 ** -10)
        oracle.close(held, y, step + 2 * near, f"{case} out8")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size", SIZES)
def test_rms_norm_of_every_width(dtype, size):
    dt = TYPES[dtype]
    for rows, with_residual in ((1, True), (37, False), (5, True)):
        print(f"rms_norm {rows} x {size} {dtype} residual {with_residual}", flush=True)
        x, gamma = cpu_randn(size, rows, size, scale=3.0, dtype=dt), 1 + 0.1 * cpu_randn(size + 1, size, dtype=FP32)
        residual = cpu_randn(size + 2, rows, size, dtype=dt) if with_residual else None
        rooms = dict(sum=Room(rows, size, dt), out=Room(rows, size, dt), out8=Room(rows, size, E4M3), scales=Room(rows, -(-size // 128), FP32))
        ok(capi.RmsNorm(placed(x), gamma.cuda(), EPS, residual=placed(residual) if with_residual else None, **{k: r.view for k, r in rooms.items()}))
        check_norm(f"{rows} x {size}", x, residual, gamma, *(rooms[k].view for k in ("sum", "out", "out8", "scales")))
        for k, r in rooms.items():
            r.untouched(k)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("size,pad,offset", [(64, 3, 1), (130, 5, 3), (1024, 8, 8), (1024, 1, 1), (4096, 7, 5), (96, 0, 1)])
def test_rms_norm_of_rows_on_any_address(dtype, size, pad, offset):
    dt, rows, ld = TYPES[dtype], 21, size + pad
    x, residual = cpu_randn(1, rows, size, dtype=dt), cpu_randn(2, rows, size, dtype=dt)
    rooms = dict(sum=Room(rows, size, dt, ld, offset), out=Room(rows, size, dt, ld, offset), out8=Room(rows, size, E4M3, ld, offset),
                 scales=Room(rows, -(-size // 128), FP32, -(-size // 128) + pad, offset))
    ok(capi.RmsNorm(placed(x, ld, offset), None, EPS, residual=placed(residual, ld, offset), **{k: r.view for k, r in rooms.items()}))
    check_norm(f"{size}", x, residual, None, *(rooms[k].view for k in ("sum", "out", "out8", "scales")))
    for k, r in rooms.items():
        r.untouched(k)


def test_rms_norm_in_place_of_its_inputs():
    x, residual, gamma = cpu_randn(1, 50, 300), cpu_randn(2, 50, 300), 1 + 0.1 * cpu_randn(3, 300, dtype=FP32)
    gx, gr = placed(x), placed(residual)
    ok(capi.RmsNorm(gx, gamma.cuda(), EPS, residual=gr, sum=gr, out=gx))
    check_norm("in place", x, residual, gamma, gr, gx, None, None)


def test_rms_norm_results_one_by_one():
    x, residual = cpu_randn(1, 9, 256), cpu_randn(2, 9, 256)
    s = Room(9, 256, BF16)
    ok(capi.RmsNorm(placed(x), None, EPS, residual=placed(residual), sum=s.view))
    check_norm("sum alone", x, residual, None, s.view, None, None, None)
    q, scales = Room(9, 256, E4M3), Room(9, 2, FP32)
    ok(capi.RmsNorm(placed(x), None, EPS, out8=q.view, scales=scales.view))
    check_norm("8 bits alone", x, None, None, None, None, q.view, scales.view)


def test_rms_norm_of_zeros_infinities_and_no_numbers():
    x = cpu_randn(1, 6, 260, dtype=FP32)
    x[0] = 0.0
    x[1, 130:] = 0.0      # a block of zeros beside others
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] *= 1e-18         # squares far below eps
    out, q, scales = Room(6, 260, FP32), Room(6, 260, E4M3), Room(6, 3, FP32)
    ok(capi.RmsNorm(x.cuda(), None, EPS, out=out.view, out8=q.view, scales=scales.view))
    _, y = oracle.rms_norm(x, None, EPS)
    assert bool(torch.isnan(out.view[2]).all()) and bool(torch.isnan(scales.view[2]).all()) and bool(torch.isnan(q.view[2].float()).all())
    assert bool(torch.isnan(out.view[3, 7])) and bool((out.view[3, :7] == 0).all())
    for row in (0, 1, 4, 5):
        pick = lambda t: t[row:row + 1]  # noqa: E731
        check_norm(f"row {row}", pick(x), None, None, None, pick(out.view), pick(q.view), pick(scales.view))
    assert bool((scales.view[0] == 2.0 ** -126).all()) and float(scales.view[1, 2]) == 2.0 ** -126 and bool((q.view[0].float() == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,size", [(1, 1), (1, 128), (3, 7), (300, 64), (5000, 128), (2100, 129), (700, 256), (33, 512), (1030, 1000), (77, 2051), (64, 4096),
                                       (9, 8200), (4, 16384)])
def test_rms_norm_backward(dtype, rows, size):
    dt = TYPES[dtype]
    for with_sum in (False, True):
        print(f"rms_norm_backward {rows} x {size} {dtype} grad_sum {with_sum}", flush=True)
        x, dy, gamma = cpu_randn(1, rows, size, scale=2.0, dtype=dt), cpu_randn(2, rows, size, dtype=dt), 1 + 0.1 * cpu_randn(3, size, dtype=FP32)
        ds = cpu_randn(4, rows, size, dtype=dt) if with_sum else None
        dx, dgamma = Room(rows, size, dt), Room(1, size, FP32)
        call = capi.RmsNormBackward(placed(x), gamma.cuda(), placed(dy), EPS, grad_sum=placed(ds) if with_sum else None, grad_x=dx.view,
                                    grad_gamma=dgamma.view[0])
        ok(call)
        want, off, want_gamma, off_gamma = oracle.rms_norm_backward(x, gamma, dy, EPS, ds)
        oracle.close(dx.view, want, oracle.stored(want, off, dt), "grad_x")
        oracle.close(dgamma.view[0], want_gamma, off_gamma + 2.0 ** -24 * want_gamma.abs(), "grad_gamma")
        dx.untouched("grad_x"), dgamma.untouched("grad_gamma")
        first = dx.view.clone(), dgamma.view.clone()
        ok(call)
        assert torch.equal(first[0], dx.view) and torch.equal(first[1], dgamma.view), "other bits the second time"


def test_rms_norm_backward_on_any_address_and_in_place():
    rows, size, ld = 40, 130, 137
    x, dy, ds, gamma = cpu_randn(1, rows, size), cpu_randn(2, rows, size), cpu_randn(3, rows, size), 1 + 0.1 * cpu_randn(4, size, dtype=FP32)
    want, off, want_gamma, off_gamma = oracle.rms_norm_backward(x, gamma, dy, EPS, ds)
    grad = placed(ds, ld, 3)
    ok(capi.RmsNormBackward(placed(x, ld, 1), gamma.cuda(), placed(dy, ld, 5), EPS, grad_sum=grad, grad_x=grad))
    oracle.close(grad, want, oracle.stored(want, off, BF16), "grad_x over grad_sum")
    dgamma = torch.empty(size, device="cuda")
    ok(capi.RmsNormBackward(placed(x, ld, 1), gamma.cuda(), placed(dy, ld, 5), EPS, grad_gamma=dgamma))
    oracle.close(dgamma, want_gamma, off_gamma + 2.0 ** -24 * want_gamma.abs(), "grad_gamma alone")


# few enough rows for a workgroup alone, which writes dgamma itself: on any address, and not past its end
@pytest.mark.parametrize("rows,size", [(1, 5), (3, 130), (4, 1999), (8, 1024), (7, 600), (16, 509), (100, 40), (2, 8193), (2, 16384)])
def test_rms_norm_backward_of_few_rows(rows, size):
    x, dy, gamma = cpu_randn(1, rows, size), cpu_randn(2, rows, size), 1 + 0.1 * cpu_randn(4, size, dtype=FP32)
    want, off, want_gamma, off_gamma = oracle.rms_norm_backward(x, gamma, dy, EPS, None)
    dx, dgamma = Room(rows, size, BF16), Room(1, size, FP32, size, 1)
    ok(capi.RmsNormBackward(x.cuda(), gamma.cuda(), dy.cuda(), EPS, grad_x=dx.view, grad_gamma=dgamma.view.view(size)))
    oracle.close(dx.view, want, oracle.stored(want, off, BF16), "grad_x")
    oracle.close(dgamma.view.view(size), want_gamma, off_gamma + 2.0 ** -24 * want_gamma.abs(), "grad_gamma")
    dx.untouched("grad_x"), dgamma.untouched("grad_gamma")


def test_rms_norm_backward_against_differences():
    rows, size, step = 3, 40, 1e-6
    x, dy, gamma = cpu_randn(1, rows, size, dtype=FP32), cpu_randn(2, rows, size, dtype=FP32), 1 + 0.1 * cpu_randn(3, size, dtype=FP32)
    dx, dgamma = torch.empty(rows, size, device="cuda"), torch.empty(size, device="cuda")
    ok(capi.RmsNormBackward(x.cuda(), gamma.cuda(), dy.cuda(), EPS, grad_x=dx, grad_gamma=dgamma))

    def loss(x64, gamma64):
        return float((x64 / torch.sqrt((x64 * x64).mean(1, keepdim=True) + EPS) * gamma64 * dy.double()).sum())

    for at in range(0, rows * size, 7):  # central differences in 64 bits: off by about step^2 and 1e-16 / step
        e = torch.zeros(rows * size, dtype=torch.float64)
        e[at] = step
        e = e.view(rows, size)
        slope = (loss(x.double() + e, gamma.double()) - loss(x.double() - e, gamma.double())) / (2 * step)
        assert abs(slope - float(dx.view(-1)[at])) < 1e-5 * (1 + abs(slope)), at
    for at in range(0, size, 5):
        e = torch.zeros(size, dtype=torch.float64)
        e[at] = step
        slope = (loss(x.double(), gamma.double() + e) - loss(x.double(), gamma.double() - e)) / (2 * step)
        assert abs(slope - float(dgamma[at])) < 1e-5 * (1 + abs(slope)), at


# ---- 8 bits ----

@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,size,pad,offset", [(1, 1, 0, 0), (1, 128, 0, 0), (130, 257, 0, 0), (128, 1024, 0, 0), (129, 96, 5, 3), (300, 4100, 0, 0), (17, 640, 3, 1)])
def test_quantiser_gives_the_definitions_bits(dtype, block_rows, rows, size, pad, offset):
    dt = TYPES[dtype]
    x = cpu_randn(rows + size, rows, size, scale=5.0, dtype=dt)
    x[0, 0] = 128.0  # a block whose quotients 448 k / 128 often lie half way between two of e4m3's
    blocks = -(-size // 128)
    q, scales = Room(rows, size, E4M3, size + pad, offset), Room(-(-rows // block_rows), blocks, FP32, blocks + pad, offset)
    ok(capi.QuantizeFp8(placed(x, size + pad, offset), q.view, scales.view, block_rows))
    want_q, want_s = oracle.quantise(x, block_rows)
    assert torch.equal(scales.view.cpu(), want_s)
    assert torch.equal(q.view.cpu().float(), want_q.float())
    q.untouched("out"), scales.untouched("scales")


def test_quantiser_far_from_one():
    x = cpu_randn(1, 8, 256, dtype=FP32)
    x[0] *= 1e-30
    x[1] *= 1e30
    x[2] *= 1e-42
    x[3] = 0.0
    x[4, 3] = math.inf
    x[5, 200] = math.nan
    q, scales = torch.empty(8, 256, device="cuda", dtype=E4M3), torch.empty(8, 2, device="cuda")
    ok(capi.QuantizeFp8(x.cuda(), q, scales))
    want_q, want_s = oracle.quantise(x, 1)
    for got, want in ((scales.cpu(), want_s), (q.cpu().float(), want_q.float())):
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def eight_bits(seed, m, n, k):
    a, a_scales = oracle.quantise(cpu_randn(seed, m, k, dtype=FP32), 1)
    w, w_scales = oracle.quantise(cpu_randn(seed + 1, n, k, scale=k ** -0.5, dtype=FP32), 128)
    return a, a_scales, w, w_scales


@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (1, 500, 4096), (2, 130, 300), (5, 8, 1024), (16, 256, 512), (17, 257, 129), (33, 64, 2000), (64, 384, 640), (65, 100, 16),
                                   (127, 129, 255), (128, 128, 128), (200, 328, 1040), (300, 1160, 2000), (512, 256, 384), (513, 515, 517), (256, 512, 8192)])
def test_linear_fp8(out, m, n, k):
    dt = TYPES[out]
    a, a_scales, w, w_scales = eight_bits(m + n + k, m, n, k)
    for bias in (None, cpu_randn(5, n, dtype=FP32)):
        print(f"linear_fp8 {m} x {n} x {k} {out} bias {bias is not None}", flush=True)
        room = Room(m, n, dt)
        ok(capi.LinearFp8(a.cuda(), a_scales.cuda(), w.cuda(), w_scales.cuda(), room.view, bias=None if bias is None else bias.cuda()))
        want, off = oracle.linear_fp8(a, a_scales, w, w_scales, bias, dt)
        oracle.close(room.view, want, oracle.stored(want, off, dt), f"{m} x {n} x {k}")
        room.untouched("out")


# enough 128 x 128 and 256 x 256 tiles for kernels of their own: ragged sides, a cut last block, several spans of scales, one block alone
@pytest.mark.parametrize("out,m,n,k", [("bf16", 1700, 1500, 2448), ("fp32", 1700, 1500, 2448), ("bf16", 1793, 1409, 112), ("fp32", 1665, 1537, 144), ("bf16", 2900, 4100, 1168),
                                       ("bf16", 3329, 3841, 96), ("bf16", 3400, 3800, 128), ("bf16", 23000, 130, 256)])
def test_linear_fp8_of_many_rows(out, m, n, k):
    dt = TYPES[out]
    a, a_scales, w, w_scales = eight_bits(m + n + k, m, n, k)
    room = Room(m, n, dt)
    ok(capi.LinearFp8(a.cuda(), a_scales.cuda(), w.cuda(), w_scales.cuda(), room.view))
    want, off = oracle.linear_fp8(a, a_scales, w, w_scales, None, dt)
    oracle.close(room.view, want, oracle.stored(want, off, dt), f"{m} x {n} x {k}")
    room.untouched("out")


@pytest.mark.parametrize("m,n,k,pad,offset", [(3, 200, 256, 16, 16), (3, 200, 256, 5, 3), (40, 130, 300, 1, 1), (150, 260, 512, 16, 0), (150, 260, 512, 7, 9)])
def test_linear_fp8_of_rows_on_any_address(m, n, k, pad, offset):
    a, a_scales, w, w_scales = eight_bits(9, m, n, k)
    blocks = -(-k // 128)
    room = Room(m, n, BF16, n + pad, offset)
    ok(capi.LinearFp8(placed(a, k + pad, offset), placed(a_scales, blocks + pad, offset), placed(w, k + pad, offset), placed(w_scales, blocks + pad, offset), room.view))
    want, off = oracle.linear_fp8(a, a_scales, w, w_scales, dtype=BF16)
    oracle.close(room.view, want, oracle.stored(want, off, BF16), "out")
    room.untouched("out")


# rows that are no whole 16-byte pieces, in tiles: several spans of scales, one cut block alone, rows of fewer than 16 bytes, a last block of one value
@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("m,n,k,pad,offset", [(1700, 1500, 2441, 0, 0), (1280, 1100, 7, 0, 0), (1300, 1410, 120, 3, 5), (1201, 1153, 257, 0, 0), (1290, 1164, 384, 1, 0), (1290, 1164, 256, 0, 8),
                                              (9900, 120, 645, 0, 1)])
def test_linear_fp8_of_many_rows_on_any_address(out, m, n, k, pad, offset):
    dt = TYPES[out]
    a, a_scales, w, w_scales = eight_bits(m + n + k, m, n, k)
    bias = cpu_randn(5, n, dtype=FP32)
    room = Room(m, n, dt, n + pad)
    ok(capi.LinearFp8(placed(a, k + pad, offset), a_scales.cuda(), placed(w, k + pad, offset), w_scales.cuda(), room.view, bias=bias.cuda()))
    want, off = oracle.linear_fp8(a, a_scales, w, w_scales, bias, dt)
    oracle.close(room.view, want, oracle.stored(want, off, dt), f"{m} x {n} x {k}")
    room.untouched("out")


# rows of fewer than 16 bytes, of 16 and 17, and a cut block that begins within one; in every form that few rows have
@pytest.mark.parametrize("out", ["bf16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(1, 300, 15), (3, 9000, 15), (3, 9000, 17), (16, 8200, 143), (9, 70, 18), (40, 3000, 130), (300, 1100, 129), (700, 900, 19), (30, 70, 2049)])
def test_linear_fp8_of_few_rows_on_any_address(out, m, n, k):
    dt = TYPES[out]
    a, a_scales, w, w_scales = eight_bits(m + n + k, m, n, k)
    room = Room(m, n, dt)
    ok(capi.LinearFp8(placed(a, k + 1, 3), a_scales.cuda(), placed(w, None, 1), w_scales.cuda(), room.view))
    want, off = oracle.linear_fp8(a, a_scales, w, w_scales, None, dt)
    oracle.close(room.view, want, oracle.stored(want, off, dt), f"{m} x {n} x {k}")
    room.untouched("out")


def test_linear_fp8_of_rows_far_apart():
    m, n, k, ld = 18, 130, 300, (1 << 23) + 16
    a, a_scales, w, w_scales = eight_bits(4, m, n, k)
    memory = torch.zeros(m, ld, device="cuda", dtype=torch.uint8).view(a.dtype)
    memory[:, :k] = a.cuda()
    room = Room(m, n, FP32)
    ok(capi.LinearFp8(memory[:, :k], a_scales.cuda(), w.cuda(), w_scales.cuda(), room.view))
    want, off = oracle.linear_fp8(a, a_scales, w, w_scales)
    oracle.close(room.view, want, oracle.stored(want, off, FP32), "out")


@pytest.mark.parametrize("m", [3, 200])
def test_linear_fp8_keeps_a_bad_row_to_itself(m):
    """A row of no numbers, and one with an infinite scale, beside others."""
    a, a_scales, w, w_scales = eight_bits(3, m, 140, 300)
    a_bytes = a.view(torch.uint8)
    a_bytes[0, 17] = 0x7F  # e4m3's not-a-number
    a_scales[1, 2] = math.inf
    out = torch.empty(m, 140, device="cuda")
    ok(capi.LinearFp8(a.cuda(), a_scales.cuda(), w.cuda(), w_scales.cuda(), out))
    want, off = oracle.linear_fp8(a[2:], a_scales[2:], w, w_scales)
    assert bool(torch.isnan(out[0]).all()) and not bool(torch.isfinite(out[1]).any())
    oracle.close(out[2:], want, oracle.stored(want, off, FP32), "the other rows")


# ---- gated transition ----

WIDTHS = [(1, 1), (8, 8), (32, 64), (64, 256), (128, 512), (128, 96), (128, 64), (256, 1024), (256, 448), (200, 328), (77, 130), (130, 2), (384, 512), (520, 1030), (512, 2048)]


def weights_of(seed, c_o, c_i):
    return cpu_randn(seed, c_i, c_o, scale=c_o ** -0.5), cpu_randn(seed + 1, c_i, c_o, scale=c_o ** -0.5), cpu_randn(seed + 2, c_o, c_i, scale=c_i ** -0.5)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("c_o,c_i", WIDTHS)
def test_gated_transition(activation, c_o, c_i):
    w = weights_of(c_o + c_i, c_o, c_i)
    gpu = [t.cuda() for t in w]
    for rows in (1, 4, 17, 33, 64, 130, 300):
        print(f"gated_transition {rows} rows {c_o} -> {c_i} {activation}", flush=True)
        x = cpu_randn(rows, rows, c_o)
        room = Room(rows, c_o, BF16)
        ok(capi.GatedTransition(x.cuda(), *gpu, room.view, activation))
        want, off = oracle.gated_transition(x, *w, activation)["out"]
        oracle.close(room.view, want, oracle.stored(want, off, BF16), f"{rows} rows {c_o} -> {c_i}")
        room.untouched("out")


@pytest.mark.parametrize("rows,c_o,c_i,pad,offset", [(3, 128, 512, 8, 8), (3, 128, 512, 3, 1), (70, 128, 256, 8, 0), (70, 128, 256, 1, 5), (300, 256, 512, 8, 0), (40, 96, 200, 7, 3)])
def test_gated_transition_of_rows_on_any_address(rows, c_o, c_i, pad, offset):
    w = weights_of(5, c_o, c_i)
    x, dy = cpu_randn(1, rows, c_o), cpu_randn(2, rows, c_o)
    gpu = [placed(t.reshape(1, -1), None, offset).view(t.shape) for t in w]  # dense, but on any address
    want = oracle.gated_transition(x, *w, "silu", dy)
    room = Room(rows, c_o, BF16, c_o + pad, offset)
    ok(capi.GatedTransition(placed(x, c_o + pad, offset), *gpu, room.view))
    oracle.close(room.view, want["out"][0], oracle.stored(*want["out"], BF16), "out")
    room.untouched("out")
    grads = [Room(rows, c_o, BF16, c_o + pad, offset), Room(c_i, c_o, BF16), Room(c_i, c_o, BF16), Room(c_o, c_i, BF16)]
    ok(capi.GatedTransitionBackward(placed(x, c_o + pad, offset), *gpu, placed(dy, c_o + pad, offset), *(r.view for r in grads)))
    for name, r in zip(("grad_x", "grad_gate_w", "grad_up_w", "grad_down_w"), grads):
        oracle.close(r.view, want[name][0], oracle.stored(*want[name], BF16), name)
        r.untouched(name)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("c_o,c_i", WIDTHS)
def test_gated_transition_backward(activation, c_o, c_i):
    w = weights_of(c_o + c_i, c_o, c_i)
    gpu = [t.cuda() for t in w]
    for rows in (1, 5, 33, 130, 700):
        print(f"gated_transition_backward {rows} rows {c_o} -> {c_i} {activation}", flush=True)
        x, dy = cpu_randn(rows, rows, c_o), cpu_randn(rows + 1, rows, c_o)
        want = oracle.gated_transition(x, *w, activation, dy)
        grads = dict(grad_x=Room(rows, c_o, BF16), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
        call = capi.GatedTransitionBackward(x.cuda(), *gpu, dy.cuda(), activation=activation, **{k: r.view for k, r in grads.items()})
        ok(call)
        for name, r in grads.items():
            oracle.close(r.view, want[name][0], oracle.stored(*want[name], BF16), f"{name} of {rows} rows {c_o} -> {c_i}")
            r.untouched(name)
        first = [r.view.clone() for r in grads.values()]
        ok(call)
        assert all(torch.equal(a, r.view) for a, r in zip(first, grads.values())), "other bits the second time"


# enough tiles for the kernels of 128, 192 and 256 rows a tile in every product: ragged sides, k that ends within a stage, an odd number of stages for two groups
@pytest.mark.parametrize("rows,c_o,c_i", [(4001, 264, 2816), (5000, 136, 2816), (8090, 2048, 72), (8090, 1032, 200), (4001, 72, 4096), (130, 1024, 4096), (2100, 512, 520), (1000, 1024, 1096),
                                          (40000, 64, 136),
                                          # ... and of widths that are no whole pieces, split by rows and by hidden units, odd ones and of few columns
                                          (5088, 124, 130), (2113, 77, 131), (1500, 515, 1030), (70, 70, 1001), (1100, 9, 4100), (3000, 1027, 12)])
def test_gated_transition_of_many_tiles(rows, c_o, c_i):
    w = weights_of(rows, c_o, c_i)
    gpu, x, dy = [t.cuda() for t in w], cpu_randn(1, rows, c_o), cpu_randn(2, rows, c_o)
    want = oracle.gated_transition(x, *w, "silu", dy)
    out = Room(rows, c_o, BF16)
    ok(capi.GatedTransition(x.cuda(), *gpu, out.view))
    oracle.close(out.view, want["out"][0], oracle.stored(*want["out"], BF16), "out")
    out.untouched("out")
    grads = dict(grad_x=Room(rows, c_o, BF16), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
    ok(capi.GatedTransitionBackward(x.cuda(), *gpu, dy.cuda(), **{k: r.view for k, r in grads.items()}))
    for name, r in grads.items():
        oracle.close(r.view, want[name][0], oracle.stored(*want[name], BF16), name)
        r.untouched(name)


# the hidden layer on chip: fewer waves than a round, several rounds with a ragged last one, one slice of hidden units and several, strided rows
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,c_o,c_i,pad", [(1, 64, 32, 0), (45, 64, 96, 8), (65, 64, 32, 0), (109, 64, 96, 8), (33000, 64, 64, 0), (8200, 128, 32, 0), (8191, 128, 64, 8), (9001, 128, 512, 0), (70001, 128, 96, 0),
                                              (20500, 256, 32, 0), (20900, 256, 160, 8), (33000, 256, 64, 0)])
def test_gated_transition_on_chip(activation, rows, c_o, c_i, pad):
    w = weights_of(rows, c_o, c_i)
    x = cpu_randn(1, rows, c_o)
    room = Room(rows, c_o, BF16, c_o + pad)
    ok(capi.GatedTransition(placed(x, c_o + pad), *(t.cuda() for t in w), room.view, activation))
    want, off = oracle.gated_transition(x, *w, activation)["out"]
    oracle.close(room.view, want, oracle.stored(want, off, BF16), "out")
    room.untouched("out")


# rows that fill no block of 32, one block a split and several, hidden units that fill no group of 128, strided rows, splits with fewer blocks than the others
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,c_o,c_i,pad", [(1, 64, 32, 0), (31, 128, 32, 8), (32, 64, 256, 0), (65, 128, 160, 8), (2049, 64, 96, 0), (9001, 128, 256, 16), (8191, 64, 320, 0), (12289, 128, 512, 0),
                                              (33001, 128, 288, 8), (70001, 64, 64, 0)])
def test_gated_transition_backward_on_chip(activation, rows, c_o, c_i, pad):
    w = weights_of(rows, c_o, c_i)
    gpu, x, dy = [t.cuda() for t in w], cpu_randn(1, rows, c_o), cpu_randn(2, rows, c_o)
    want = oracle.gated_transition(x, *w, activation, dy)
    grads = dict(grad_x=Room(rows, c_o, BF16, c_o + pad), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
    call = capi.GatedTransitionBackward(placed(x, c_o + pad), *gpu, placed(dy, c_o + 2 * pad), activation=activation, **{k: r.view for k, r in grads.items()})
    ok(call)
    for name, r in grads.items():
        oracle.close(r.view, want[name][0], oracle.stored(*want[name], BF16), name)
        r.untouched(name)
    first = [r.view.clone() for r in grads.values()]
    ok(call)
    assert all(torch.equal(a, r.view) for a, r in zip(first, grads.values())), "other bits the second time"
    for name, r in grads.items():  # each alone
        room = Room(*r.view.shape, BF16)
        ok(capi.GatedTransitionBackward(placed(x, c_o + pad), *gpu, placed(dy, c_o + 2 * pad), activation=activation, **{name: room.view}))
        assert torch.equal(room.view, r.view), name
        room.untouched(name)


# up to 64 rows: one block of 32 and two, full and not; fewer channels than waves share, and as many as the LDS holds
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("rows,c_o,c_i,pad", [(1, 2048, 96, 0), (64, 1024, 1024, 8), (63, 96, 32, 0), (32, 32, 32, 8), (33, 32, 64, 0), (17, 1056, 160, 16), (64, 2048, 32, 0), (2, 160, 4096, 0)])
def test_gated_transition_backward_of_few_rows(activation, rows, c_o, c_i, pad):
    w = weights_of(rows, c_o, c_i)
    gpu, x, dy = [t.cuda() for t in w], cpu_randn(1, rows, c_o), cpu_randn(2, rows, c_o)
    want = oracle.gated_transition(x, *w, activation, dy)
    grads = dict(grad_x=Room(rows, c_o, BF16, c_o + pad), grad_gate_w=Room(c_i, c_o, BF16), grad_up_w=Room(c_i, c_o, BF16), grad_down_w=Room(c_o, c_i, BF16))
    ok(capi.GatedTransitionBackward(placed(x, c_o + pad), *gpu, placed(dy, c_o + 2 * pad), activation=activation, **{k: r.view for k, r in grads.items()}))
    for name, r in grads.items():
        oracle.close(r.view, want[name][0], oracle.stored(*want[name], BF16), name)
        r.untouched(name)
        room = Room(*r.view.shape, BF16)  # and alone
        ok(capi.GatedTransitionBackward(placed(x, c_o + pad), *gpu, placed(dy, c_o + 2 * pad), activation=activation, **{name: room.view}))
        assert torch.equal(room.view, r.view), name


@pytest.mark.parametrize("rows", [40, 90])
def test_gated_transition_backward_keeps_a_bad_row_to_itself(rows):
    """In the gradient of x; the weights' gradients are not-a-number where the sum over the rows is, the last row's included where its block of 32 is not full."""
    c_o, c_i = 128, 256
    w = weights_of(1, c_o, c_i)
    x, dy = cpu_randn(1, rows, c_o), cpu_randn(2, rows, c_o)
    dy[rows - 1, 5] = math.nan
    grads = [Room(rows, c_o, BF16), Room(c_i, c_o, BF16), Room(c_i, c_o, BF16), Room(c_o, c_i, BF16)]
    ok(capi.GatedTransitionBackward(x.cuda(), *(t.cuda() for t in w), dy.cuda(), *(r.view for r in grads)))
    want = oracle.gated_transition(x[:-1], *w, "silu", dy[:-1])
    assert bool(torch.isnan(grads[0].view[-1]).all())
    oracle.close(grads[0].view[:-1], want["grad_x"][0], oracle.stored(*want["grad_x"], BF16), "the other rows")
    assert bool(torch.isnan(grads[1].view).all()) and bool(torch.isnan(grads[2].view).all()) and bool(torch.isnan(grads[3].view[5]).all())
    others = [c for c in range(c_o) if c != 5]
    want = oracle.gated_transition(x, *w, "silu", torch.nan_to_num(dy))
    oracle.close(grads[3].view[others], want["grad_down_w"][0][others], oracle.stored(*want["grad_down_w"], BF16)[others], "the other channels of Wd")


def test_gated_transition_backward_gives_the_gradients_that_are_asked_for():
    rows, c_o, c_i = 90, 128, 192
    w = weights_of(1, c_o, c_i)
    gpu, x, dy = [t.cuda() for t in w], cpu_randn(1, rows, c_o), cpu_randn(2, rows, c_o)
    want = oracle.gated_transition(x, *w, "silu", dy)
    for name, shape in (("grad_x", (rows, c_o)), ("grad_gate_w", (c_i, c_o)), ("grad_up_w", (c_i, c_o)), ("grad_down_w", (c_o, c_i))):
        room = Room(*shape, BF16)
        ok(capi.GatedTransitionBackward(x.cuda(), *gpu, dy.cuda(), **{name: room.view}))
        oracle.close(room.view, want[name][0], oracle.stored(*want[name], BF16), name)
        room.untouched(name)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gated_transition_of_large_values(activation):
    """Gates far on both sides of zero: the sigmoid ends at 0 and 1, its derivative at 0."""
    rows, c_o, c_i = 40, 128, 128
    w = weights_of(1, c_o, c_i)
    gpu, x, dy = [t.cuda() for t in w], cpu_randn(1, rows, c_o, scale=300.0), cpu_randn(2, rows, c_o)
    want = oracle.gated_transition(x, *w, activation, dy)
    out, grads = Room(rows, c_o, BF16), [Room(rows, c_o, BF16), Room(c_i, c_o, BF16), Room(c_i, c_o, BF16), Room(c_o, c_i, BF16)]
    ok(capi.GatedTransition(x.cuda(), *gpu, out.view, activation))
    oracle.close(out.view, want["out"][0], oracle.stored(*want["out"], BF16), "out")
    ok(capi.GatedTransitionBackward(x.cuda(), *gpu, dy.cuda(), *(r.view for r in grads), activation=activation))
    for name, r in zip(("grad_x", "grad_gate_w", "grad_up_w", "grad_down_w"), grads):
        oracle.close(r.view, want[name][0], oracle.stored(*want[name], BF16), name)


# few results, whose hidden layer keeps what its rounding leaves: a rounding within 2^-8 of a rest within 2^-8 of the value, in place of the first alone
@pytest.mark.parametrize("rows,c_o,c_i", [(1, 128, 512), (16, 256, 520), (17, 64, 256), (64, 64, 128), (1, 4096, 64), (2, 2048, 72), (33, 120, 1000)])
def test_gated_transition_of_few_results_rounds_once(rows, c_o, c_i):
    w = weights_of(rows, c_o, c_i)
    x = cpu_randn(1, rows, c_o)
    out = torch.empty(rows, c_o, device="cuda", dtype=BF16)
    ok(capi.GatedTransition(x.cuda(), *(t.cuda() for t in w), out))
    want, off = oracle.gated_transition(x, *w, "silu")["out"]
    h = torch.nn.functional.silu(x.double() @ w[0].double().T) * (x.double() @ w[1].double().T)
    off = off - (2.0 ** -8 - 2.0 ** -16) * (h.abs() @ w[2].double().abs().T)
    assert bool((off > 0).all())
    oracle.close(out, want, oracle.stored(want, off, BF16), "out")


@pytest.mark.parametrize("rows,c_o,c_i", [(40, 128, 256), (40, 96, 160)])
def test_gated_transition_keeps_a_bad_row_to_itself(rows, c_o, c_i):
    w = weights_of(1, c_o, c_i)
    x = cpu_randn(1, rows, c_o)
    x[0, 3], x[rows - 1, 5] = math.nan, math.inf
    out = torch.empty(rows, c_o, device="cuda", dtype=BF16)
    ok(capi.GatedTransition(x.cuda(), *(t.cuda() for t in w), out))
    want, off = oracle.gated_transition(x[1:-1], *w, "silu")["out"]
    assert bool(torch.isnan(out[0]).all()) and not bool(torch.isfinite(out[-1]).any())
    oracle.close(out[1:-1], want, oracle.stored(want, off, BF16), "the other rows")


# ---- as they are used ----

def test_a_block_in_training_end_to_end():
    """sum = x + residual, y = norm(sum), out = sum + transition(y); gradients of x, gamma and the weights against 64-bit autograd."""
    rows, c, c_i = 150, 128, 384
    x, residual, gamma, dy = cpu_randn(1, rows, c), cpu_randn(2, rows, c), 1 + 0.1 * cpu_randn(3, c, dtype=FP32), cpu_randn(4, rows, c)
    w = weights_of(5, c, c_i)
    gpu, gx, gr, gg, gdy = [t.cuda() for t in w], x.cuda(), residual.cuda(), gamma.cuda(), dy.cuda()
    s, y, out = (torch.empty(rows, c, device="cuda", dtype=BF16) for _ in range(3))
    ok(capi.RmsNorm(gx, gg, EPS, residual=gr, sum=s, out=y))
    ok(capi.GatedTransition(y, *gpu, out))
    grads = [torch.empty_like(t) for t in (y, *gpu)]
    ok(capi.GatedTransitionBackward(y, *gpu, gdy, *grads))
    dx, dgamma = torch.empty_like(y), torch.empty_like(gg)
    ok(capi.RmsNormBackward(s, gg, grads[0], EPS, grad_sum=gdy, grad_x=dx, grad_gamma=dgamma))

    leaves = [t.double().requires_grad_() for t in (x, gamma, *w)]
    s64 = leaves[0] + residual.double()
    y64 = s64 / torch.sqrt((s64 * s64).mean(1, keepdim=True) + EPS) * leaves[1]
    f64 = (torch.nn.functional.silu(y64 @ leaves[2].T) * (y64 @ leaves[3].T)) @ leaves[4].T
    (s64 + f64).backward(dy.double())
    # y, s, h, dg, du, the gradient of y and each result are rounded to bf16 in a chain of at most five, each within 2^-8 of its values: in the
    # 2-norm 5 x 2^-8 together, where no step multiplies relative errors (condition about 1 for these weights; 2 leaves room)
    for name, got, want in [("out", out, f64), ("grad_x", dx, leaves[0].grad), ("grad_gamma", dgamma, leaves[1].grad)] + [
            (f"weight {i}", g, t.grad) for i, (g, t) in enumerate(zip(grads[1:], leaves[2:]))]:
        rel = float((got.cpu().double() - want.detach()).norm() / want.detach().norm())
        assert rel < 2 * 5 * 2.0 ** -8, (name, rel)


def test_a_projection_in_8_bits_behind_its_norm():
    """The operand that the norm writes is the one that the product takes; weights from the quantiser."""
    for rows in (1, 70, 260):
        c, n = 320, 200
        x, residual, gamma, weight = cpu_randn(1, rows, c), cpu_randn(2, rows, c), 1 + 0.1 * cpu_randn(3, c, dtype=FP32), cpu_randn(4, n, c, scale=c ** -0.5)
        s, q, scales = torch.empty(rows, c, device="cuda", dtype=BF16), torch.empty(rows, c, device="cuda", dtype=E4M3), torch.empty(rows, 3, device="cuda")
        w, w_scales, out = torch.empty(n, c, device="cuda", dtype=E4M3), torch.empty(2, 3, device="cuda"), torch.empty(rows, n, device="cuda", dtype=BF16)
        ok(capi.QuantizeFp8(weight.cuda(), w, w_scales, 128))
        ok(capi.RmsNorm(x.cuda(), gamma.cuda(), EPS, residual=residual.cuda(), sum=s, out8=q, scales=scales))
        ok(capi.LinearFp8(q, scales, w, w_scales, out))
        want, off = oracle.linear_fp8(q, scales, w, w_scales, dtype=BF16)
        oracle.close(out, want, oracle.stored(want, off, BF16), f"{rows} rows")
        # and it is the product of what went in: 8 bits on either side are within 2^-4 of their values, 2^-4.5 on average at most
        _, y = oracle.rms_norm(x, gamma, EPS, residual)
        plain = y @ weight.double().T
        assert float((out.cpu().double() - plain).norm() / plain.norm()) < 2 * 2.0 ** -4


def operators_of_everything(rows, c, c_i, seed):
    """One call of each operator, and the tensors that they write."""
    w = [t.cuda() for t in weights_of(seed, c, c_i)]
    x, residual, dy, gamma = (cpu_randn(seed + i, rows, c).cuda() for i in (3, 4, 5)), None, None, None
    x, residual, dy = x
    gamma = 1 + 0.1 * cpu_randn(seed + 6, c, dtype=FP32).cuda()
    e = lambda *shape, dtype=BF16: torch.zeros(*shape, device="cuda", dtype=FP32).to(dtype)  # noqa: E731
    s, y, q, scales = e(rows, c), e(rows, c), e(rows, c, dtype=E4M3), e(rows, -(-c // 128), dtype=FP32)
    w8, w8_scales, product = e(c_i, c, dtype=E4M3), e(-(-c_i // 128), -(-c // 128), dtype=FP32), e(rows, c_i)
    out, dx, dgamma, grads = e(rows, c), e(rows, c), e(c, dtype=FP32), [e(rows, c), e(c_i, c), e(c_i, c), e(c, c_i)]
    calls = [capi.RmsNorm(x, gamma, EPS, residual=residual, sum=s, out=y, out8=q, scales=scales), capi.QuantizeFp8(w[0], w8, w8_scales, 128),
             capi.LinearFp8(q, scales, w8, w8_scales, product), capi.GatedTransition(y, *w, out),
             capi.GatedTransitionBackward(y, *w, dy, *grads), capi.RmsNormBackward(s, gamma, grads[0], EPS, grad_sum=dy, grad_x=dx, grad_gamma=dgamma)]
    results = [s, y, q, scales, w8, w8_scales, product, out, dx, dgamma, *grads]
    return calls, results, x


def run_all(calls, stream=None):
    for call in calls:
        rc = call.run(stream)
        assert rc == 0, (type(call).__name__, rc)


@pytest.mark.parametrize("rows,c,c_i", [(3, 512, 1024), (700, 128, 512), (400, 384, 640), (100, 64, 128), (13000, 128, 512), (200, 131, 259)])
def test_captured_and_replayed(rows, c, c_i):
    calls, results, x = operators_of_everything(rows, c, c_i, 1)
    run_all(calls)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run_all(calls, torch.cuda.current_stream().cuda_stream)
    for seed in (10, 11, 12):
        x.copy_(cpu_randn(seed, rows, c).cuda())
        for r in results:
            r.view(torch.uint8).zero_()
        run_all(calls)
        torch.cuda.synchronize()
        want = [r.view(torch.uint8).clone() for r in results]
        for r in results:
            r.view(torch.uint8).fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, r.view(torch.uint8)) for a, r in zip(want, results)), f"replay {seed}"


def test_two_at_once_on_streams_of_their_own():
    sets = [operators_of_everything(300, 128, 512, 1), operators_of_everything(500, 256, 768, 20)]
    want = []
    for calls, results, _ in sets:
        run_all(calls)
        torch.cuda.synchronize()
        want.append([r.view(torch.uint8).clone() for r in results])
        for r in results:
            r.view(torch.uint8).zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for (calls, _, _), stream in zip(sets, streams):
            run_all(calls, stream.cuda_stream)
    torch.cuda.synchronize()
    for (_, results, _), w in zip(sets, want):
        assert all(torch.equal(a, r.view(torch.uint8)) for a, r in zip(w, results))


@pytest.mark.parametrize("c", [128, 127])
def test_more_elements_than_32_bits_count(c):
    """The first and the last rows of calls whose operands end past 2^31 elements; the gradient of out is zero but in the last ones."""
    c_i, last = 32, 40
    rows = (1 << 31) // c + 3 * last
    w, gamma = weights_of(7, c, c_i), 1 + 0.1 * cpu_randn(3, c, dtype=FP32)
    gpu, x_last, dy_last = [t.cuda() for t in w], cpu_randn(1, last, c), cpu_randn(2, last, c)
    x, dy = torch.zeros(rows, c, device="cuda", dtype=BF16), torch.zeros(rows, c, device="cuda", dtype=BF16)
    x[:last], x[-last:], dy[-last:] = x_last.cuda(), x_last.cuda(), dy_last.cuda()
    out, grads = torch.ones_like(x), [torch.empty_like(t) for t in gpu]

    def check(got, want, dtype, what):
        oracle.close(got, want[0], oracle.stored(want[0], want[1], dtype), what)

    want = oracle.gated_transition(x_last, *w, "silu", dy_last)
    ok(capi.GatedTransition(x, *gpu, out))
    check(out[:last], want["out"], BF16, "the first rows")
    check(out[-last:], want["out"], BF16, "the last rows")
    assert not bool(out[last:-last].any())
    ok(capi.GatedTransitionBackward(x, *gpu, dy, out, *grads))
    check(out[-last:], want["grad_x"], BF16, "grad_x")
    assert not bool(out[:-last].any())
    for name, g in zip(("grad_gate_w", "grad_up_w", "grad_down_w"), grads):
        check(g, want[name], BF16, name)

    s64, y64 = oracle.rms_norm(x_last, gamma, EPS)
    out8, scales = torch.empty(rows, c, device="cuda", dtype=E4M3), torch.empty(rows, 1, device="cuda")
    ok(capi.RmsNorm(x, gamma.cuda(), EPS, out=out, out8=out8, scales=scales))
    near = [torch.empty(last, c, device="cuda", dtype=t.dtype) for t in (out, out8)] + [torch.empty(last, 1, device="cuda")]
    ok(capi.RmsNorm(x_last.cuda(), gamma.cuda(), EPS, out=near[0], out8=near[1], scales=near[2]))
    for a, b in zip((out, out8, scales), near):
        assert torch.equal(a[:last].view(torch.uint8), b.view(torch.uint8)) and torch.equal(a[-last:].view(torch.uint8), b.view(torch.uint8))
    dgamma, want_dgamma = torch.empty(c, device="cuda"), torch.empty(c, device="cuda")
    near_dx = torch.empty(last, c, device="cuda", dtype=BF16)
    ok(capi.RmsNormBackward(x, gamma.cuda(), dy, EPS, grad_x=out, grad_gamma=dgamma))
    ok(capi.RmsNormBackward(x_last.cuda(), gamma.cuda(), dy_last.cuda(), EPS, grad_x=near_dx, grad_gamma=want_dgamma))
    assert torch.equal(out[-last:], near_dx) and not bool(out[:-last].any())
    # sums of 40 products, in two orders
    bound = 2 * 40 * oracle.ADD * (dy_last.double().abs() * y64.abs() / gamma.double().abs()).sum(0) * (1 + 2 ** -10)
    assert bool(((dgamma - want_dgamma).double().cpu().abs() <= bound).all())

    w8, w_scales = torch.empty(24, c, device="cuda", dtype=E4M3), torch.empty(1, 1, device="cuda")
    ok(capi.QuantizeFp8(cpu_randn(9, 24, c).cuda(), w8, w_scales, 128))
    product, near_product = torch.empty(rows, 24, device="cuda", dtype=BF16), torch.empty(last, 24, device="cuda", dtype=BF16)
    ok(capi.LinearFp8(out8, scales, w8, w_scales, product))
    ok(capi.LinearFp8(near[1], near[2], w8, w_scales, near_product))
    want, off = oracle.linear_fp8(near[1].cpu(), near[2].cpu(), w8.cpu(), w_scales.cpu(), None, BF16)
    for got in (product[:last], product[-last:], near_product):
        check(got, (want, off), BF16, "product")


def test_calls_of_no_rows_do_nothing():
    e = lambda *shape, dtype=BF16: torch.zeros(*shape, device="cuda", dtype=FP32).to(dtype)  # noqa: E731
    w = [t.cuda() for t in weights_of(1, 64, 128)]
    ok(capi.RmsNorm(e(0, 64), None, EPS, out=e(0, 64)))
    ok(capi.QuantizeFp8(e(0, 64), e(0, 64, dtype=E4M3), e(0, 1, dtype=FP32)))
    ok(capi.LinearFp8(e(0, 64, dtype=E4M3), e(0, 1, dtype=FP32), e(8, 64, dtype=E4M3), e(1, 1, dtype=FP32), e(0, 8)))
    ok(capi.GatedTransition(e(0, 64), *w, e(0, 64)))
