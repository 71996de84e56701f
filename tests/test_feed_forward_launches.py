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
    far = record([transition(rows, c_o, c_i, backward) for rows, c_o in shapes for backward in (False, True) for c_i in (limit, (1 << 30) - 64)])
    for r in near:
        assert r.rc == 0 and not any("ff_tiles_kernel" in k.kernel for k in r.launches), r
    for r in far:
        assert r.rc == 0 and any("ff_tiles_kernel" in k.kernel for k in r.launches), r
        pitched = [k for k in r.launches if ("ff_pieces_kernel" in k.kernel or "ff_split_kernel" in k.kernel)]
        # the first product of the forward pass alone, whose operands' rows are c_o apart
        assert all("kernelILi1E" in k.kernel for k in pitched) and len(pitched) <= 1, r
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
