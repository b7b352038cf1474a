"""Sizes of the serving operators' C ABI whose products leave 64 bits, on the CPU."""

from __future__ import annotations

import ctypes

import pytest

UNSUPPORTED = 2


def _cache():
    from robustgemq_b200._lib import KvCacheT

    c = KvCacheT()
    c.k = c.v = 0x10000
    c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.bits, c.dtype = 8, 4, 16, 128, 16, 0
    c.strides = (4 * 16 * 256, 16 * 256, 256)
    return ctypes.byref(c)


@pytest.mark.parametrize("tokens", [(1 << 29) + 1, 1 << 62, (1 << 62) + 4, (1 << 63) - 4])
def test_token_counts_that_wrap(tokens):
    """Four heads times 2^62 tokens is 0 in 64 bits."""
    from robustgemq_b200 import _lib

    lib = _lib.load()
    assert lib.gemq_kv_cache_write(_cache(), 0x1000, 0x1000, 512, 128, 512, 128, 0x1000, tokens, None) == UNSUPPORTED
    assert lib.gemq_kv_cache_read(_cache(), 0x1000, tokens, 0x1000, 0x1000, None) == UNSUPPORTED
    assert lib.gemq_paged_attention_workspace_size(_cache(), tokens, 4, 4, 8, 0, 0) == 0
    assert lib.gemq_paged_attention(_cache(), 0x1000, 512, tokens, 4, 0x1000, 8, 8, 0x1000, None, 4, 0, 0, 1.0, 0, 0x1000,
                                    None, None, 0, None) == UNSUPPORTED
