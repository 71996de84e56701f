"""Which kernels the feed-forward calls take, with what grids and LDS; without a GPU."""
from kutacc_amd import capi
from recorded_launches import AT, record

BF16 = capi.K_BF16


def transition(rows, c_o, c_i, backward=False, **over):
    fields = dict(rows=rows, c_o=c_o, c_i=c_i, dtype=BF16, activation=0, x=AT, x_ld=c_o, gate_w=AT, up_w=AT, down_w=AT, workspace=AT, workspace_bytes=1 << 50)
    fields.update(dict(grad_out=AT, grad_out_ld=c_o, grad_x=AT, grad_x_ld=c_o, grad_gate_w=AT, grad_up_w=AT, grad_down_w=AT) if backward else dict(out=AT, out_ld=c_o))
    fields.update(over)
    return (f"kutacc_hip_gated_transition{'_backward' if backward else ''}", f"HipGatedTransition{'Backward' if backward else ''}Args", fields)


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
