"""Which kernels the feed-forward calls take, with what grids and LDS; without a GPU."""
from kutacc_amd import capi
from recorded_launches import AT, record

BF16, FP32 = capi.K_BF16, capi.K_FP32


def transition(rows, c_o, c_i, backward=False, **over):
    fields = dict(rows=rows, c_o=c_o, c_i=c_i, dtype=BF16, activation=0, x=AT, x_ld=c_o, gate_w=AT, up_w=AT, down_w=AT, workspace=AT, workspace_bytes=1 << 50)
    fields.update(dict(grad_out=AT, grad_out_ld=c_o, grad_x=AT, grad_x_ld=c_o, grad_gate_w=AT, grad_up_w=AT, grad_down_w=AT) if backward else dict(out=AT, out_ld=c_o))
    fields.update(over)
    return (f"kutacc_hip_gated_transition{'_backward' if backward else ''}", f"HipGatedTransition{'Backward' if backward else ''}Args", fields)


def linear(m, n, k, out=BF16, **over):
    blocks = -(-k // 128)
    fields = dict(m=m, n=n, k=k, dtype=out, a=AT, a_ld=k, a_scales=AT, a_scales_ld=blocks, w=AT, w_ld=k, w_scales=AT, w_scales_ld=blocks, out=AT, out_ld=n)
    return "kutacc_hip_linear_fp8", "HipLinearFp8Args", {**fields, **over}


# The kernels of whole pieces count bytes from a tile's first row in 32 bits: not where rows of the hidden layer, of down_w or of the operands are 2^23 elements apart
def test_far_apart_rows_take_the_kernels_that_count_in_64_bits():
    limit = 1 << 23
    shapes = [(1, 8), (32, 8), (128, 72), (300, 256), (20000, 136)]
    near = record([transition(rows, c_o, limit - 32, backward) for rows, c_o in shapes for backward in (False, True)])
    far = record([transition(rows, c_o, c_i, backward) for rows, c_o in shapes for backward in (False, True) for c_i in (limit, (1 << 30) - 64) if rows * c_i <= 1 << 38])
    for r in near:
        assert r.rc == 0 and not any("ff_tiles_kernel" in k.kernel for k in r.launches), r
    for r in far:
        assert r.rc == 0 and any("ff_tiles_kernel" in k.kernel for k in r.launches), r
        assert not any("ff_pieces_kernel" in k.kernel or "ff_split_kernel" in k.kernel for k in r.launches), r
    wide = record([transition(300, limit, 64, backward) for backward in (False, True)] + [transition(300, 256, 512, backward, x_ld=limit) for backward in (False, True)])
    for r in wide:
        assert r.rc == 0 and any("ff_tiles_kernel" in k.kernel for k in r.launches), r


# A kernel is opted into dynamic LDS once: with a size of its own for every width, a later call would have to do it in a capture, or two threads' first calls could leave it
# with the smaller of theirs
def test_kernels_are_opted_into_their_lds_once():
    shapes = [(rows, c_o, c_i) for rows in (1, 20, 33, 64, 300, 20000) for c_o in (32, 64, 128, 256, 1024, 2048) for c_i in (32, 64, 512, 1056)]
    calls = [transition(*shape, backward, activation=act) for shape in shapes for backward in (False, True) for act in (0, 1)]
    calls += [linear(m, n, k, out) for m in (1, 16, 40, 300, 5000) for n in (64, 1000, 8192) for k in (100, 128, 4096) for out in (BF16, FP32)]
    sizes = {}
    for r in record(calls):
        assert r.rc == 0, r
        for kernel, size in r.opted:
            sizes.setdefault(kernel, set()).add(size)
        for k in r.launches:
            assert k.lds <= max(sizes.get(k.kernel, {64 << 10})) <= 160 << 10, k
    assert len(sizes) > 10 and all(len(s) == 1 for s in sizes.values()), {k: s for k, s in sizes.items() if len(s) > 1}


def norm(rows, size, dtype=BF16):
    fields = dict(rows=rows, size=size, dtype=dtype, eps=1e-6, x=AT, x_ld=size, residual=AT, residual_ld=size, sum=AT, sum_ld=size, out=AT, out_ld=size, out8=AT, out8_ld=size,
                  scales=AT, scales_ld=-(-size // 128))
    return "kutacc_hip_rms_norm", "HipRmsNormArgs", fields


def quantise(rows, size, block_rows):
    return "kutacc_hip_quantize_fp8", None, [AT, size, AT, size, AT, -(-size // 128), rows, size, block_rows, BF16]


# A launch has fewer than 2^32 threads: calls with work for more are made in parts or with larger tiles, or refused before anything of them is launched
def test_no_launch_has_2_to_the_32_threads():
    rows = [1 << 20, (1 << 27) + 5, (1 << 28) + 1, (1 << 29) + 1, (1 << 30) - 1]
    calls = [norm(r, size, dtype) for r in rows + [1 << 23, (1 << 33) + 7] for size in (1, 64, 65, 128, 513, 16384) for dtype in (BF16, FP32) if r * size <= 1 << 37]
    calls += [quantise(r, size, block) for r in rows + [100, (1 << 33) + 7] for size in (1, 64, 129, 5000, 1 << 29) for block in (1, 128) if r * size <= 1 << 37]
    calls += [transition(r, c_o, c_i, backward) for r in rows for c_o in (8, 32, 64, 77, 128, 256, 264) for c_i in (8, 32, 64, 77) for backward in (False, True)
              if r * (2 * c_o + (c_i + 31) // 32 * 32) <= 1 << 37]
    calls += [transition(1, 8, c_i, backward) for c_i in ((1 << 23) - 32, 1 << 24, 1 << 27, (1 << 30) - 32, (1 << 30) - 1) for backward in (False, True)]
    taken = record(calls)
    for c, r in zip(calls, taken):
        assert r.rc == 0, (c, r)
    refused = [linear((1 << 30) - 1, 1, 15), linear(1, (1 << 30) - 1, 16), linear(1, 1 << 29, 128, FP32)]
    for c, r in zip(refused, record(refused)):
        assert r.rc == capi.EUNSUPPORTED and not r.launches, (c, r)
    lines = [linear(m, n, k, out) for m, n in (((1 << 30) - 1, 8), (1 << 26, 300), (1, 1 << 26), (16, 1 << 28), (300, 1 << 26)) for k in (16, 17, 128) for out in (BF16, FP32)]
    taken += record(lines)
    for r in taken:
        assert r.rc == 0 and r.launches, r
        for k in r.launches:
            assert k.grid[1:] == (1, 1) and 0 < k.grid[0] < 1 << 31 and k.grid[0] * k.threads < 1 << 32, (r, k)


def test_parts_of_a_call_are_all_of_it():
    for rows, size, per_group in (((1 << 29) + 1, 64, 32), ((1 << 33) + 7, 128, 16), ((1 << 28) + 9, 512, 4)):
        (r,) = record([norm(rows, size)])
        whole = (2 ** 32 - 1) // 256 * per_group
        assert [k.grid[0] for k in r.launches] == [(min(rows - at, whole) + per_group - 1) // per_group for at in range(0, rows, whole)]
    rows = (1 << 33) + 7
    (a, w) = record([quantise(rows, 200, 1), quantise(rows, 200, 128)])
    whole = (2 ** 32 - 1) // 256 * 16 // 2
    assert [k.grid[0] for k in a.launches] == [-(-min(rows - at, whole) * 2 // 16) for at in range(0, rows, whole)]
    whole = (2 ** 32 - 1) // 256 // 2 * 128
    assert [k.grid[0] for k in w.launches] == [-(-min(rows - at, whole) // 128) * 2 for at in range(0, rows, whole)]
