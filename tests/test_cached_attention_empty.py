"""Calls of nothing: tensors of no element, which have no address, and sequences of no token.  The library's part runs without a GPU."""
import pytest
import torch

from kutacc_amd import capi
from test_cached_attention_host import append, attention, rotary


def test_no_tokens_and_no_addresses():
    assert rotary(tokens=0, q__data=None, q_out__data=None, k__data=None, k_out__data=None) == 0
    assert rotary(tokens=4, q__data=None, q_out__data=None, k__data=None, k_out__data=None) == capi.EINVAL
    none = dict(batch__tokens=0, q__data=None)
    assert append(**none, q_out__data=None, k__data=None, v__data=None) == 0
    assert attention(**none, out__data=None, lse=None) == (0, 0)


@pytest.mark.gpu
def test_owners_of_nothing():
    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    inv_freq = capi.rotary_frequencies(64).cuda()
    int32 = torch.int32
    cache = capi.Cache(empty(3, 16, 2, 64), empty(3, 16, 2, 64))
    for sequences in (0, 2):
        batch = capi.CacheBatch(torch.zeros(sequences + 1, dtype=int32, device="cuda"), torch.zeros(sequences, dtype=int32, device="cuda"), empty(sequences, 1, dtype=int32))
        assert capi.Rotary(empty(0, 4, 64), inv_freq, k=empty(0, 2, 64)).run() == 0
        assert capi.CacheAppend(cache, batch, empty(0, 2, 64), empty(0, 2, 64), inv_freq, q=empty(0, 4, 64)).run() == 0
        assert capi.CachedAttention(cache, batch, empty(0, 4, 64), empty(0, 4, 64), lse=empty(0, 4, dtype=torch.float32)).run() == 0
    torch.cuda.synchronize()
