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
