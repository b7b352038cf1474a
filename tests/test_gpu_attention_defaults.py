"""Paged attention, and the cache, called as plainly as they can be: hints left out, and
tensors that lie as another layer left them."""

from __future__ import annotations

import pytest
import torch

from serving_helpers import Batch

pytestmark = pytest.mark.gpu
H16, B16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    from robustgemq_b200 import _lib

    _lib.device_error()
    yield
    assert _lib.device_error() == 0


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("each", [1, 4])
@pytest.mark.parametrize("max_q_len", [0, 1, 1000])
def test_without_starts_a_batch_of_few_tokens_takes_its_own_kernel(bits, each, max_q_len):
    """As many tokens a sequence as there are for it, whatever the hint says: the kernel for
    few rows, by its bits (the one for chunks sums in another order)."""
    from robustgemq_b200.serving import paged_attention

    b = Batch([(each, 100 + 37 * i) for i in range(64)], 8, 1, 128, 16, bits, H16)
    want = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts, max_q_len=each)
    got = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, max_q_len=max_q_len)
    assert torch.equal(got, want)
    b.check(use_starts=False, max_q_len=max_q_len)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("n", [1, 50])
def test_queries_and_rows_that_start_off_16_bytes(bits, n):
    """Contiguous tensors that begin anywhere in a buffer, and one token with a row stride
    that is no multiple of 8."""
    from robustgemq_b200.serving import paged_attention

    b = Batch([(n, 90)], 4, 2, 64, 16, bits, H16)
    want, _ = b.check()
    for off in (1, 3, 8):
        buf = torch.zeros(b.q.numel() + 16, dtype=H16, device="cuda")
        q = buf[off:off + b.q.numel()].view_as(b.q)
        q.copy_(b.q)
        assert q.is_contiguous()
        assert torch.equal(paged_attention(q, b.cache, b.page_table, b.kv_lens), want)
        k = torch.randn((n, 2, 64), device="cuda").half()
        rows = buf[off:off + k.numel()].view_as(k)
        rows.copy_(k)
        slots = b.slots(0, torch.arange(n, device="cuda"))
        b.cache.write(k, k, slots)
        first = b.cache.read(slots)
        b.cache.write(torch.zeros_like(k), torch.zeros_like(k), slots)
        b.cache.write(rows, rows, slots)
        assert all(torch.equal(x, y) for x, y in zip(b.cache.read(slots), first))
        b = Batch([(n, 90)], 4, 2, 64, 16, bits, H16)
    if n == 1:
        wide = torch.zeros((1, 4 * 64 + 3), dtype=H16, device="cuda")
        wide[:, :256] = b.q.view(1, 256)
        q = wide.as_strided((1, 4, 64), (259, 64, 1))
        assert torch.equal(paged_attention(q, b.cache, b.page_table, b.kv_lens), want)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_caches_whose_axes_of_one_element_have_other_strides(bits):
    """One page, K from a pool and V of its own: the strides between pages say nothing."""
    from robustgemq_b200.serving import PagedKVCache

    own = PagedKVCache(1, 16, 2, 64, bits=bits)
    pool = torch.zeros((1, 3, *own.k.shape[1:]), dtype=own.k.dtype, device="cuda")
    scales = () if bits == 16 else (torch.zeros((1, 5, *own.k_scale.shape[1:]), device="cuda")[:, 2], own.v_scale)
    cache = PagedKVCache.from_tensors(pool[:, 1], own.v, *scales, dtype=H16)
    x, y = (torch.randn((16, 2, 64), device="cuda").half() for _ in range(2))
    slots = torch.arange(16, device="cuda")
    cache.write(x, y, slots)
    own.write(x, y, slots)
    for got, want in zip(cache.read(slots), own.read(slots)):
        assert torch.equal(got, want)
