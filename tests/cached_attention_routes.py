"""Which form cached attention takes, found from what it wants as its workspace; without a GPU it answers as for a device of 256 CUs."""
import ctypes

from kutacc_amd import capi


def _sizes(page_size, kv_heads, head_size, sequences, tokens, columns, prefix, heads):
    a = capi.HipCachedAttentionArgs()
    a.cache.pages, a.cache.page_size, a.cache.kv_heads, a.cache.head_size, a.cache.dtype = 1, page_size, kv_heads, head_size, capi.K_BF16
    a.batch.sequences, a.batch.tokens, a.batch.columns, a.batch.prefix_length, a.q_heads = sequences, tokens, columns, prefix, heads
    return capi.lib().kutacc_hip_cached_attention_workspace(ctypes.byref(a))


def prefix_is_shared(page_size, kv_heads, head_size, sequences, tokens, columns, prefix, heads):
    """Whether the prefix is read once for the batch, by workgroups of its own.  Otherwise a call wants the workspace of one whose sequences have the prefix among their own entries."""
    if prefix == 0:
        return False
    one = (kv_heads, head_size, sequences, tokens)
    return _sizes(page_size, *one, columns, prefix, heads) != _sizes(1, *one, columns * page_size + prefix, 0, heads)
