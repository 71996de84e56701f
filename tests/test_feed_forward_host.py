"""What the feed-forward entry points refuse, before anything is launched: these run without a GPU."""
import ctypes

import pytest

from kutacc_amd import capi

AT = 1 << 32  # an address that nothing reads


def norm(**over):
    a = capi.HipRmsNormArgs()
    fields = dict(rows=4, size=256, dtype=capi.K_BF16, eps=1e-6, x=AT, x_ld=256, residual=AT, residual_ld=256, gamma=AT, sum=AT, sum_ld=256, out=AT, out_ld=256,
                  out8=AT, out8_ld=256, scales=AT, scales_ld=2)
    for k, v in {**fields, **over}.items():
        setattr(a, k, v)
    return capi.lib().kutacc_hip_rms_norm(ctypes.byref(a), None)


@pytest.mark.parametrize("over", [dict(rows=-1), dict(size=0), dict(size=-5), dict(dtype=0), dict(dtype=3), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(x_ld=255),
                                  dict(residual_ld=255), dict(sum_ld=0), dict(out_ld=255), dict(out8_ld=100), dict(scales_ld=1), dict(scales=None),
                                  dict(out8=None), dict(out=None, out8=None, scales=None, sum=None)])
def test_rms_norm_refuses(over):
    assert norm(**over) == capi.EINVAL


def test_rms_norm_says_what_it_has_no_kernel_for():
    wide = dict(size=16385, x_ld=1 << 15, residual_ld=1 << 15, sum_ld=1 << 15, out_ld=1 << 15, out8_ld=1 << 15, scales_ld=256)
    assert norm(**wide) == capi.EUNSUPPORTED
    assert norm(rows=0) == 0
    assert capi.lib().kutacc_hip_rms_norm(None, None) == capi.EINVAL


def norm_backward(**over):
    a = capi.HipRmsNormBackwardArgs()
    fields = dict(rows=4, size=256, dtype=capi.K_BF16, eps=1e-6, x=AT, x_ld=256, gamma=AT, grad_out=AT, grad_out_ld=256, grad_sum=AT, grad_sum_ld=256, grad_x=AT,
                  grad_x_ld=256, grad_gamma=AT, workspace=AT, workspace_bytes=1 << 20)
    for k, v in {**fields, **over}.items():
        setattr(a, k, v)
    return capi.lib().kutacc_hip_rms_norm_backward(ctypes.byref(a), None)


@pytest.mark.parametrize("over", [dict(rows=0), dict(rows=-1), dict(size=0), dict(dtype=7), dict(eps=-1.0), dict(x=None), dict(x_ld=255), dict(grad_out=None), dict(grad_out_ld=1),
                                  dict(grad_sum_ld=1), dict(grad_x_ld=255), dict(grad_x=None, grad_gamma=None), dict(workspace=None), dict(workspace=AT + 16),
                                  dict(workspace_bytes=1023)])
def test_rms_norm_backward_refuses(over):
    assert norm_backward(**over) == capi.EINVAL


def test_rms_norm_backward_says_what_it_has_no_kernel_for():
    wide = dict(size=16385, x_ld=1 << 15, grad_out_ld=1 << 15, grad_sum_ld=1 << 15, grad_x_ld=1 << 15)
    assert norm_backward(**wide) == capi.EUNSUPPORTED
    L = capi.lib()
    assert L.kutacc_hip_rms_norm_backward_workspace(4, 256) >= 1024 and L.kutacc_hip_rms_norm_backward_workspace(-1, 256) == capi.EINVAL
    assert L.kutacc_hip_rms_norm_backward_workspace(4, 0) == capi.EINVAL and L.kutacc_hip_rms_norm_backward(None, None) == capi.EINVAL


def quantise(x=AT, x_ld=256, out=AT, out_ld=256, scales=AT, scales_ld=2, rows=4, size=256, block_rows=1, dtype=capi.K_BF16):
    return capi.lib().kutacc_hip_quantize_fp8(x, x_ld, out, out_ld, scales, scales_ld, rows, size, block_rows, dtype, None)


@pytest.mark.parametrize("over", [dict(x=None), dict(x_ld=255), dict(out=None), dict(out_ld=255), dict(scales=None), dict(scales_ld=1), dict(rows=-1), dict(size=0),
                                  dict(block_rows=0), dict(block_rows=64), dict(dtype=0)])
def test_quantiser_refuses(over):
    assert quantise(**over) == capi.EINVAL


def linear(**over):
    a = capi.HipLinearFp8Args()
    fields = dict(m=4, n=300, k=256, dtype=capi.K_BF16, a=AT, a_ld=256, a_scales=AT, a_scales_ld=2, w=AT, w_ld=256, w_scales=AT, w_scales_ld=2, bias=AT, out=AT, out_ld=300)
    for k, v in {**fields, **over}.items():
        setattr(a, k, v)
    return capi.lib().kutacc_hip_linear_fp8(ctypes.byref(a), None)


@pytest.mark.parametrize("over", [dict(m=-1), dict(n=0), dict(k=0), dict(m=1 << 31), dict(n=1 << 31), dict(k=1 << 31), dict(dtype=0), dict(a=None), dict(a_ld=255), dict(a_scales=None),
                                  dict(a_scales_ld=1), dict(w=None), dict(w_ld=255), dict(w_scales=None), dict(w_scales_ld=1), dict(out=None), dict(out_ld=299)])
def test_linear_fp8_refuses(over):
    assert linear(**over) == capi.EINVAL


def transition(backward, **over):
    a = capi.HipGatedTransitionBackwardArgs() if backward else capi.HipGatedTransitionArgs()
    fields = dict(rows=300, c_o=96, c_i=130, dtype=capi.K_BF16, activation=0, x=AT, x_ld=96, gate_w=AT, up_w=AT, down_w=AT, workspace=AT, workspace_bytes=1 << 30)
    more = dict(grad_out=AT, grad_out_ld=96, grad_x=AT, grad_x_ld=96, grad_gate_w=AT, grad_up_w=AT, grad_down_w=AT) if backward else dict(out=AT, out_ld=96)
    for k, v in {**fields, **more, **over}.items():
        setattr(a, k, v)
    L = capi.lib()
    return (L.kutacc_hip_gated_transition_backward if backward else L.kutacc_hip_gated_transition)(ctypes.byref(a), None)


BOTH = [dict(rows=-1), dict(rows=1 << 31), dict(c_o=0), dict(c_i=0), dict(dtype=capi.K_FP32), dict(dtype=0), dict(activation=2), dict(activation=-1), dict(x=None), dict(x_ld=95),
        dict(gate_w=None), dict(up_w=None), dict(down_w=None), dict(workspace=None), dict(workspace=AT + 128), dict(workspace_bytes=1000)]


@pytest.mark.parametrize("over", BOTH + [dict(out=None), dict(out_ld=95)])
def test_gated_transition_refuses(over):
    assert transition(False, **over) == capi.EINVAL


@pytest.mark.parametrize("over", BOTH + [dict(rows=0), dict(grad_out=None), dict(grad_out_ld=95), dict(grad_x_ld=95),
                                         dict(grad_x=None, grad_gate_w=None, grad_up_w=None, grad_down_w=None)])
def test_gated_transition_backward_refuses(over):
    assert transition(True, **over) == capi.EINVAL


def test_workspaces_of_what_is_no_shape():
    L = capi.lib()
    for f in (L.kutacc_hip_gated_transition_workspace, L.kutacc_hip_gated_transition_backward_workspace):
        assert f(-1, 8, 8) == f(1, 0, 8) == f(1, 8, 0) == f(1 << 31, 8, 8) == capi.EINVAL and f(0, 8, 8) == 0
    assert transition(False, rows=0) == 0 and linear(m=0) == 0 and quantise(rows=0) == 0
    assert L.kutacc_hip_gated_transition(None, None) == L.kutacc_hip_gated_transition_backward(None, None) == L.kutacc_hip_linear_fp8(None, None) == capi.EINVAL
