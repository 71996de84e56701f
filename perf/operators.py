"""The operators of a feed-forward half of a transformer block, each as a user's program calls it and in plain form.

  op             entry point
  norm           kutacc_hip_rms_norm: residual addition and RMS norm, results in storage type and/or 8 bits with scales
  norm_backward  kutacc_hip_rms_norm_backward
  linear_fp8     kutacc_hip_linear_fp8: product of 8-bit operands with a scale for each block of 128; `quantise`: with
                 kutacc_hip_quantize_fp8 of the activation in front of it
  ff             kutacc_hip_gated_transition: out = (act(x gate^T) * (x up^T)) down^T
  ff_backward    kutacc_hip_gated_transition_backward: gradients of x and of the three weights
"""
import math

import torch

own = False

EPS = 1e-6
BLOCK = 128          # values that share a scale
LARGEST = 448.0      # of e4m3
SMALLEST_SCALE = 2.0 ** -126
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # Eight sequences decoding one token each: the norm in front of 8-bit projections, where latency is all there is.
        dict(name="norm_fp8_8x4096", op="norm", dtype="bf16", rows=8, size=4096, residual=True, plain=False, fp8=True),
        # A batch of prompts, a row short of a whole number of tiles, normalised into 8 bits with its residual stream kept.
        dict(name="norm_fp8_8191x4096", op="norm", dtype="bf16", rows=8191, size=4096, residual=True, plain=False, fp8=True),
        # The pair activation of 384 residues in training: short rows, very many of them.
        dict(name="norm_backward_147456x128", op="norm_backward", dtype="bf16", rows=384 * 384, size=128, residual=True),
        # fp32 training of an odd width, whose rows start on any multiple of four bytes.
        dict(name="norm_backward_fp32_1021x2051", op="norm_backward", dtype="fp32", rows=1021, size=2051, residual=False),
        # One token through an 8-bit projection: the weights' bytes are all there is.
        dict(name="linear_fp8_1x8192x4096", op="linear_fp8", m=1, n=8192, k=4096, out="bf16", bias=False, quantise=False),
        # A large batch of prompts: the matrix cores' rate.
        dict(name="linear_fp8_8192x4096x8192", op="linear_fp8", m=8192, n=4096, k=8192, out="bf16", bias=False, quantise=False),
        # Ragged everywhere (the last blocks of k and n are cut), quantised on the way in, with a bias and an fp32 result.
        dict(name="linear_fp8_777x1160x2000", op="linear_fp8", m=777, n=1160, k=2000, out="fp32", bias=True, quantise=True),
        # Three tokens through a wide block: weights' bytes again, in bf16, and two products that depend on each other.
        dict(name="ff_3x2048x8192", op="ff", act="silu", rows=3, c_o=2048, c_i=8192),
        # The pair activation of 384 residues.
        dict(name="ff_147456x128x512", op="ff", act="silu", rows=384 * 384, c_o=128, c_i=512),
        # A ragged batch at a middle width, whose hidden width is no power of two, with the other activation.
        dict(name="ff_4001x1024x2816", op="ff", act="gelu", rows=4001, c_o=1024, c_i=2816),
        # Training: the pair activation of a crop of 256 residues ...
        dict(name="ff_backward_65536x128x512", op="ff_backward", act="silu", rows=256 * 256, c_o=128, c_i=512),
        # ... and a block of a middle width.
        dict(name="ff_backward_4096x1024x4096", op="ff_backward", act="silu", rows=4096, c_o=1024, c_i=4096),
    ]


def _size(rng, low, high):
    """A size between low and high, even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A width: mostly a multiple of 128, else a multiple of 8, now and then any number."""
    w, kind = _size(rng, low, high), rng.random()
    return max(128, w // 128 * 128) if kind < 0.5 else max(8, w // 8 * 8) if kind < 0.85 else w


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "linear_fp8", "ff", "ff_backward"])
    if op in ("norm", "norm_backward"):
        size = _width(rng, 32, 8192)
        case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp32"]), rows=_size(rng, 1, max(1, (32 << 20) // size)), size=size,
                    residual=rng.random() < 0.6)
        if op == "norm":
            kind = rng.choice(["plain", "fp8", "both"])
            case.update(plain=kind != "fp8", fp8=kind != "plain")
        return case
    if op == "linear_fp8":
        n, k = _width(rng, 64, 8192), _width(rng, 64, 8192)
        return dict(op=op, m=_size(rng, 1, max(1, min(16384, (1 << 38) // (n * k)))), n=n, k=k, out=rng.choice(["bf16", "bf16", "fp32"]),
                    bias=rng.random() < 0.4, quantise=rng.random() < 0.4)
    c_o = rng.choice([64, 128, 128, 256, 256, 384, 512, 1024, _width(rng, 32, 2048)])
    c_i = rng.choice([2 * c_o, 4 * c_o, 4 * c_o, _width(rng, 64, 8192)])
    limit = (1 << 36) // 6 if op == "ff" else (1 << 36) // 16
    return dict(op=op, act=rng.choice(["silu", "gelu"]), rows=_size(rng, 1, max(1, min(200000, limit // (c_o * c_i)))), c_o=c_o, c_i=c_i)


# ---- inputs ----

def _blocks_of(x, rows, columns):
    """x, its two axes cut into blocks of rows x columns, zeros past the end: [row blocks, rows, column blocks, columns]."""
    m, n = x.shape
    x = torch.nn.functional.pad(x, (0, -n % columns, 0, -m % rows))
    return x.view(x.shape[0] // rows, rows, x.shape[1] // columns, columns)


def _quantised(x, rows):
    """fp32 [m, n] -> e4m3 [m, n] and fp32 [ceil(m / rows), ceil(n / 128)]: the largest value of a block becomes 448."""
    b = _blocks_of(x, rows, BLOCK)
    amax = b.abs().amax((1, 3))
    scale = (amax / torch.full_like(amax, LARGEST)).clamp_min(SMALLEST_SCALE)  # a quotient: by a number, torch multiplies with its reciprocal
    q = (b / scale[:, None, :, None]).clamp(-LARGEST, LARGEST)
    q = q.reshape(b.shape[0] * rows, -1)[: x.shape[0], : x.shape[1]].contiguous()
    return q.to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    def activation(rows, size, dtype=torch.bfloat16):
        """N(0, 1) with a few channels that are ten times as large, as residual streams have."""
        channels = 1.0 + 9.0 * (torch.rand(size, device="cuda", generator=g) < 0.01)
        return (torch.randn(rows, size, device="cuda", generator=g) * channels).to(dtype)

    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, device="cuda", dtype=dtype)

    op = case["op"]
    s = dict(case=case)
    if op == "norm":
        dt, rows, size = TYPES[case["dtype"]], case["rows"], case["size"]
        s["x"] = activation(rows, size, dt)
        s["residual"] = activation(rows, size, dt) if case["residual"] else None
        s["gamma"] = 1.0 + 0.1 * torch.randn(size, device="cuda", generator=g)
        s["sum"] = empty(rows, size, dtype=dt) if case["residual"] else None
        s["out"] = empty(rows, size, dtype=dt) if case["plain"] else None
        s["out8"] = empty(rows, size, dtype=torch.float8_e4m3fn) if case["fp8"] else None
        s["scales"] = empty(rows, -(-size // BLOCK), dtype=torch.float32) if case["fp8"] else None
    elif op == "norm_backward":
        dt, rows, size = TYPES[case["dtype"]], case["rows"], case["size"]
        s["x"] = activation(rows, size, dt)
        s["gamma"] = 1.0 + 0.1 * torch.randn(size, device="cuda", generator=g)
        s["grad_out"] = normal(rows, size, dtype=dt)
        s["grad_sum"] = normal(rows, size, dtype=dt) if case["residual"] else None
        s["grad_x"], s["grad_gamma"] = empty(rows, size, dtype=dt), empty(size, dtype=torch.float32)
    elif op == "linear_fp8":
        m, n, k = case["m"], case["n"], case["k"]
        x = activation(m, k)
        if case["quantise"]:
            s["x"], s["a"] = x, empty(m, k, dtype=torch.float8_e4m3fn)
            s["a_scales"] = empty(m, -(-k // BLOCK), dtype=torch.float32)
        else:
            s["a"], s["a_scales"] = _quantised(x.float(), 1)
        s["w"], s["w_scales"] = _quantised(torch.randn(n, k, device="cuda", generator=g) * k ** -0.5, BLOCK)
        s["bias"] = 0.1 * torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        s["out"] = empty(m, n, dtype=TYPES[case["out"]])
    else:
        rows, c_o, c_i = case["rows"], case["c_o"], case["c_i"]
        s["x"] = normal(rows, c_o)
        s["gate_w"], s["up_w"] = normal(c_i, c_o, scale=c_o ** -0.5), normal(c_i, c_o, scale=c_o ** -0.5)
        s["down_w"] = normal(c_o, c_i, scale=c_i ** -0.5)
        if op == "ff":
            s["out"] = empty(rows, c_o)
        else:
            s["grad_out"] = normal(rows, c_o)
            s["grads"] = tuple(empty(*shape) for shape in ((rows, c_o), (c_i, c_o), (c_i, c_o), (c_o, c_i)))
    if own:
        s["calls"] = _calls(case, s)  # argument blocks over these tensors, and their workspaces
    return s


def _calls(case, s):
    from kutacc_amd import capi
    op = case["op"]
    if op == "norm":
        return [capi.RmsNorm(s["x"], s["gamma"], EPS, residual=s["residual"], sum=s["sum"], out=s["out"], out8=s["out8"], scales=s["scales"])]
    if op == "norm_backward":
        return [capi.RmsNormBackward(s["x"], s["gamma"], s["grad_out"], EPS, grad_sum=s["grad_sum"], grad_x=s["grad_x"], grad_gamma=s["grad_gamma"])]
    if op == "linear_fp8":
        product = capi.LinearFp8(s["a"], s["a_scales"], s["w"], s["w_scales"], s["out"], bias=s["bias"])
        return [capi.QuantizeFp8(s["x"], s["a"], s["a_scales"]), product] if case["quantise"] else [product]
    if op == "ff":
        return [capi.GatedTransition(s["x"], s["gate_w"], s["up_w"], s["down_w"], s["out"], activation=case["act"])]
    return [capi.GatedTransitionBackward(s["x"], s["gate_w"], s["up_w"], s["down_w"], s["grad_out"], *s["grads"], activation=case["act"])]


# ---- one pass ----

def run(state):
    case = state["case"]
    if own:
        for call in state["calls"]:
            rc = call.run()
            if rc != 0:
                raise RuntimeError(f"the library returned {rc}")
        op = case["op"]
        if op == "norm":
            return {k: state[k] for k in ("sum", "out", "out8", "scales")}
        if op == "norm_backward":
            return state["grad_x"], state["grad_gamma"]
        if op == "linear_fp8":
            return (state["out"], state["a"], state["a_scales"]) if case["quantise"] else (state["out"],)
        return state["out"] if op == "ff" else state["grads"]
    return {"norm": _norm, "norm_backward": _norm_backward, "linear_fp8": _linear_fp8, "ff": _ff, "ff_backward": _ff_backward}[case["op"]](state)


def _norm(s):
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["gamma"]
    q, scales = _quantised(y, 1) if s["out8"] is not None else (None, None)
    dt = s["x"].dtype
    return dict(sum=x.to(dt) if s["residual"] is not None else None, out=y.to(dt) if s["out"] is not None else None, out8=q, scales=scales)


def _norm_backward(s):
    x, dy = s["x"].float(), s["grad_out"].float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    h = dy * s["gamma"]
    dx = r * (h - x * (r * r * (h * x).mean(-1, keepdim=True)))
    if s["grad_sum"] is not None:
        dx = dx + s["grad_sum"].float()
    return dx.to(s["x"].dtype), (dy * x * r).sum(0)


def _spread(scales, rows, columns, per_row):
    """A scale for each value of a [rows, columns] operand."""
    return scales.repeat_interleave(per_row, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :columns]


def _linear_fp8(s):
    a, a_scales = (s["a"], s["a_scales"]) if not s["case"]["quantise"] else _quantised(s["x"].float(), 1)
    x = a.float() * _spread(a_scales, *a.shape, 1)
    w = s["w"].float() * _spread(s["w_scales"], *s["w"].shape, BLOCK)
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    y = y.to(s["out"].dtype)
    return (y, a, a_scales) if s["case"]["quantise"] else (y,)


def _slope(v, act):
    """What the sigmoid of the activation v * sigmoid(t(v)) is taken of, and the derivative of that."""
    if act == "silu":
        return v, torch.ones_like(v)
    c = 2.0 * math.sqrt(2.0 / math.pi)
    return c * (v + 0.044715 * v * v * v), c * (1.0 + 3.0 * 0.044715 * v * v)


def _ff(s):
    x = s["x"].float()
    g, u = x @ s["gate_w"].float().t(), x @ s["up_w"].float().t()
    h = g / (1.0 + torch.exp(-_slope(g, s["case"]["act"])[0])) * u
    return (h @ s["down_w"].float().t()).to(s["x"].dtype)


def _ff_backward(s):
    x, dy = s["x"].float(), s["grad_out"].float()
    wg, wu, wd = (s[k].float() for k in ("gate_w", "up_w", "down_w"))
    g, u, dh = x @ wg.t(), x @ wu.t(), dy @ wd
    t, slope = _slope(g, s["case"]["act"])
    sig = 1.0 / (1.0 + torch.exp(-t))
    a = g * sig
    dg, du = dh * u * (sig + a * (1.0 - sig) * slope), dh * a
    dt = s["x"].dtype
    return (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ (a * u)).to(dt)


# ---- what a pass cannot do without ----

def work(case):
    op = case["op"]
    if op == "norm":
        e, n = TYPES[case["dtype"]].itemsize, case["rows"] * case["size"]
        scales = 4 * case["rows"] * -(-case["size"] // BLOCK) if case["fp8"] else 0
        return dict(bytes=n * (e * (1 + 2 * case["residual"] + case["plain"]) + case["fp8"]) + scales + 4 * case["size"], flops=8 * n)
    if op == "norm_backward":
        e, n = TYPES[case["dtype"]].itemsize, case["rows"] * case["size"]
        return dict(bytes=n * e * (3 + case["residual"]) + 8 * case["size"], flops=12 * n)
    if op == "linear_fp8":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        return dict(bytes=m * k * (3 if case["quantise"] else 1) + n * k + 4 * (m * kb + -(-n // BLOCK) * kb + n * case["bias"])
                    + m * n * TYPES[case["out"]].itemsize, flops=2 * m * n * k)
    rows, c_o, c_i = case["rows"], case["c_o"], case["c_i"]
    if op == "ff":
        return dict(bytes=2 * (2 * rows * c_o + 3 * c_o * c_i), flops=6 * rows * c_o * c_i)
    return dict(bytes=2 * (3 * rows * c_o + 6 * c_o * c_i), flops=16 * rows * c_o * c_i)


# ---- the definitions in 64 bits ----

def exact(case, seed):
    """8-bit results before their rounding: what stands in a block over its scale."""
    s = prepare(case, seed)
    op = case["op"]

    def d(key):
        return s[key].double()

    def group_scales(y):
        rows, size = y.shape
        amax = torch.zeros(rows, -(-size // BLOCK), dtype=torch.float64, device=y.device)
        for i in range(amax.shape[1]):
            amax[:, i] = y[:, i * BLOCK:(i + 1) * BLOCK].abs().max(1).values
        return torch.maximum(amax / LARGEST, torch.tensor(SMALLEST_SCALE, dtype=torch.float64, device=y.device))

    def over(y, scales):
        return torch.cat([y[:, i * BLOCK:(i + 1) * BLOCK] / scales[:, i:i + 1] for i in range(scales.shape[1])], 1)

    if op == "norm":
        v = d("x") + (d("residual") if case["residual"] else 0.0)
        y = v / torch.sqrt((v ** 2).sum(1, keepdim=True) / case["size"] + EPS) * d("gamma")
        scales = group_scales(y) if case["fp8"] else None
        return dict(sum=v if case["residual"] else None, out=y if case["plain"] else None, out8=over(y, scales) if case["fp8"] else None,
                    scales=scales)
    if op == "norm_backward":
        v, dy = d("x"), d("grad_out")
        norm = torch.sqrt((v ** 2).sum(1, keepdim=True) / case["size"] + EPS)
        unit = v / norm
        h = dy * d("gamma")
        dx = (h - unit * (h * unit).sum(1, keepdim=True) / case["size"]) / norm + (d("grad_sum") if case["residual"] else 0.0)
        return dx, (dy * unit).sum(0)
    if op == "linear_fp8":
        if case["quantise"]:
            scales = group_scales(d("x"))
            values = over(d("x"), scales)
            # the product is of what the 8 bits hold: rounded once to 32 and then to 8, as the definition of the operand has it
            held = over(d("x"), scales.float().double()).float().to(torch.float8_e4m3fn).double()
        else:
            scales, held = d("a_scales"), d("a")
        out = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for j in range(s["w_scales"].shape[0]):  # 128 rows of weights, which share their scales
            columns = slice(j * BLOCK, min((j + 1) * BLOCK, case["n"]))
            row_scales = (scales.float().double() * s["w_scales"][j].double()).repeat_interleave(BLOCK, 1)[:, :case["k"]]
            out[:, columns] = (held * row_scales) @ s["w"][columns].double().T
        if case["bias"]:
            out += d("bias")
        return (out, values, scales) if case["quantise"] else (out,)
    x, wg, wu, wd = d("x"), d("gate_w"), d("up_w"), d("down_w")
    g, u = torch.matmul(x, wg.T), torch.matmul(x, wu.T)
    if case["act"] == "silu":
        sig = torch.sigmoid(g)
        a, da = g * sig, sig * (1 + g * (1 - sig))
    else:  # 0.5 v (1 + tanh(w))
        th = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        a = 0.5 * g * (1 + th)
        da = 0.5 * (1 + th) + 0.5 * g * (1 - th ** 2) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g ** 2)
    if op == "ff":
        return torch.matmul(a * u, wd.T)
    dy = d("grad_out")
    dh = torch.matmul(dy, wd)
    dg, du = dh * u * da, dh * a
    return torch.matmul(dg, wg) + torch.matmul(du, wu), torch.matmul(dg.T, x), torch.matmul(du.T, x), torch.matmul(dy.T, a * u)
