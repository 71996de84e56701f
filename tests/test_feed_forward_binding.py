"""What the Python owners of the feed-forward calls refuse of their tensors, on the CPU."""
import pytest
import torch

from kutacc_amd import capi

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def e(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype)


def test_rms_norm_owner_refuses_wrong_tensors():
    x = e(4, 64)
    capi.RmsNorm(x, None, out=e(4, 64))
    for bad in (dict(out=e(4, 63)), dict(out=e(4, 64, dtype=torch.float32)), dict(residual=e(64, 4).t()), dict(out8=e(4, 64)), dict(scales=e(4, 2, dtype=torch.float32)),
                dict(out=torch.empty(4, 64, dtype=BF16, device="meta"))):
        with pytest.raises(ValueError):
            capi.RmsNorm(x, None, **bad)
    with pytest.raises(ValueError):
        capi.RmsNorm(x, e(64), out=e(4, 64))  # gamma is fp32
    with pytest.raises(ValueError):
        capi.RmsNormBackward(x, None, e(4, 65), grad_x=e(4, 64))


def test_linear_owner_refuses_wrong_tensors():
    a, s, w, ws = e(4, 300, dtype=E4M3), e(4, 3, dtype=torch.float32), e(200, 300, dtype=E4M3), e(2, 3, dtype=torch.float32)
    capi.LinearFp8(a, s, w, ws, e(4, 200))
    for args in ((e(4, 300), s, w, ws, e(4, 200)), (a, e(4, 2, dtype=torch.float32), w, ws, e(4, 200)), (a, s, e(200, 301, dtype=E4M3), ws, e(4, 200)),
                 (a, s, w, e(1, 3, dtype=torch.float32), e(4, 200)), (a, s, w, ws, e(4, 201)), (a, s, w, ws, e(4, 200, dtype=torch.float16))):
        with pytest.raises((ValueError, TypeError)):
            capi.LinearFp8(*args)
    with pytest.raises(ValueError):
        capi.QuantizeFp8(e(4, 300), e(4, 300, dtype=E4M3), e(4, 2, dtype=torch.float32))


def test_transition_owner_refuses_wrong_tensors():
    x, wide, tall = e(4, 64), e(96, 64), e(64, 96)
    capi.GatedTransition(x, wide, wide, tall, e(4, 64))
    for args in ((x, wide, e(95, 64), tall, e(4, 64)), (x, wide, wide, wide, e(4, 64)), (x, wide, wide, e(96, 64).t(), e(4, 64)), (x, wide, wide, tall, e(4, 65)),
                 (x.float(), wide, wide, tall, e(4, 64))):
        with pytest.raises(ValueError):
            capi.GatedTransition(*args)
    with pytest.raises(KeyError):
        capi.GatedTransition(x, wide, wide, tall, e(4, 64), activation="relu")
    with pytest.raises(ValueError):
        capi.GatedTransitionBackward(x, wide, wide, tall, e(4, 64), grad_gate_w=tall)


def owners():
    f32 = torch.float32
    x, wide, tall, q, scales = e(4, 64), e(96, 64), e(64, 96), e(4, 64, dtype=E4M3), e(4, 1, dtype=f32)
    return [capi.RmsNorm(x, None, out=e(4, 64)), capi.RmsNormBackward(x, None, e(4, 64), grad_x=e(4, 64)), capi.QuantizeFp8(x, q, scales),
            capi.LinearFp8(q, scales, e(96, 64, dtype=E4M3), e(1, 1, dtype=f32), e(4, 96)), capi.GatedTransition(x, wide, wide, tall, e(4, 64)),
            capi.GatedTransitionBackward(x, wide, wide, tall, e(4, 64), grad_x=e(4, 64))]


def test_owners_of_host_tensors_do_not_run(monkeypatch):
    """Nothing reaches the library, which would take the addresses for a device's."""
    calls = owners()
    monkeypatch.setattr(capi, "lib", lambda: pytest.fail("the library was called"))
    for call in calls:
        with pytest.raises(ValueError, match="not the current GPU"):
            call.run()


def test_owners_run_on_their_own_device_alone(monkeypatch):
    calls = owners()
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0

    monkeypatch.setattr(capi, "lib", Library)
    for call in calls:
        call.checked_device = torch.device("cuda", 0)
        with pytest.raises(ValueError, match="cuda:0"):
            call.run()
        call.checked_device = torch.device("cuda", 1)
        assert call.run() == 0


@pytest.mark.parametrize("capturing", [False, True])
@pytest.mark.parametrize("streams", [[], [0x7000], [0x7000, 0x8000, 0x7000], [None]])
def test_a_workspace_that_goes_waits_for_its_streams(monkeypatch, streams, capturing):
    """PyTorch's allocator is told of each stream on which the call may still run, once; None is the library's own.  Streams that have finished, or are no more, it need not
    know, and none is asked during a capture."""
    told = []
    states = {0x7000: "works", 0x8000: "has finished", 0x9000: "is no more"}

    class Workspace:
        device, is_cuda = "the device", True

        def record_stream(self, stream):
            told.append(stream.ptr)

    class Stream:
        def __init__(self, ptr, device):
            assert device == "the device"
            self.ptr = ptr

        def query(self):
            assert not capturing
            if states[self.ptr] == "is no more":
                raise RuntimeError
            return states[self.ptr] == "has finished"

    class Library:
        def __getattr__(self, name):
            return lambda *args: 0x9000 if name == "kutacc_hip_get_stream" else 0

    calls = [c for c in owners() if c.workspace is not None]
    assert len(calls) == 3
    monkeypatch.setattr(capi, "lib", Library)
    monkeypatch.setattr(torch.cuda, "ExternalStream", Stream)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    while calls:
        call = calls.pop()
        call.workspace, call.checked_device = Workspace(), None
        for s in streams:
            assert call.run(s) == 0
        del call
        on = {s or 0x9000 for s in streams}
        assert sorted(told) == sorted(p for p in on if capturing or states[p] == "works")
        told.clear()
