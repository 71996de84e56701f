"""What the kernel profiler says of cached attention: how many operations a launch has is not known to the host, which knows no lengths."""
import ctypes

import pytest
import torch

from kutacc_amd import capi
from test_gpu_cached_attention import BF16, Batch, ok, randn

pytestmark = pytest.mark.gpu


def profile_of(call):
    """(name, milliseconds, launches, operations of one) of each kernel of the call."""
    lib, name = capi.lib(), ctypes.create_string_buffer(128)
    ms, launches, flops, found = ctypes.c_double(), ctypes.c_int64(), ctypes.c_double(), []
    lib.kutacc_hip_profile_enable(1)
    try:
        ok(call)
        while lib.kutacc_hip_profile_read(len(found), name, 128, ctypes.byref(ms), ctypes.byref(launches), ctypes.byref(flops)) == 0:
            found.append((name.value.decode(), ms.value, launches.value, flops.value))
    finally:
        lib.kutacc_hip_profile_enable(0)
    return found


@pytest.mark.parametrize("sequences,prefix,kernels", [([(1, 3000)], 0, 2), ([(1, 500)] * 3, 2000, 2), ([(300, 300)], 0, 1), ([(300, 300)], 70, 1)])
def test_operations_of_lengths_on_the_device_are_none(sequences, prefix, kernels):
    b = Batch(sequences, prefix, 16, 1, 64)
    cache, batch = b.on_gpu()
    call = capi.CachedAttention(cache, batch, randn(1, b.tokens, 4, 64).cuda(), torch.empty(b.tokens, 4, 64, dtype=BF16, device="cuda"))
    found = profile_of(call)
    assert [name for name, *_ in found] == ["cached_attention_kernel", "combine_kernel"][:kernels]
    assert all(ms > 0.0 and launches == 1 and flops == 0.0 for _, ms, launches, flops in found), found
