"""Attention over a paged cache with lengths and starts that no host check can see: what
they name outside the buffers is left out and recorded, and nothing else is touched."""

from __future__ import annotations

import ctypes

import pytest
import torch

from serving_helpers import Batch

pytestmark = pytest.mark.gpu
H16, B16 = torch.float16, torch.bfloat16
BAD_POSITION = 10


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    from robustgemq_b200 import _lib

    _lib.device_error()
    yield
    assert _lib.device_error() == 0


def guarded_call(b, starts, lens, table, max_q_len=0, guard=1 << 20):
    """A C ABI call whose workspace is as large as asked for; workspace and output lie
    between guards, which must stay as they are."""
    from robustgemq_b200 import _lib

    lib = _lib.load()
    cache = ctypes.cast(b.cache.c_struct, ctypes.POINTER(_lib.KvCacheT))
    seqs, tokens = lens.numel(), b.q.shape[0]
    sizes = (tokens, b.heads, seqs, table.shape[1], max_q_len, 0)
    need = lib.gemq_paged_attention_workspace_size(cache, *sizes)
    assert need > 0
    ws = torch.full((need + 2 * guard,), 0x5a, dtype=torch.uint8, device="cuda")
    out = torch.full((b.q.numel() + guard,), 7.0, dtype=b.dtype, device="cuda")
    at = guard // 2
    _lib.check(lib.gemq_paged_attention(
        cache, b.q.data_ptr(), b.q.stride(0), tokens, b.heads, table.data_ptr(), table.stride(0), table.shape[1],
        lens.data_ptr(), starts.data_ptr(), seqs, max_q_len, 0, b.dim ** -0.5, 0, out[at:].data_ptr(), None,
        ws[guard:].data_ptr(), need, _lib.stream_ptr(b.q.device)))
    torch.cuda.synchronize()
    assert (ws[:guard] == 0x5a).all() and (ws[guard + need:] == 0x5a).all()
    assert (out[:at] == 7.0).all() and (out[at + b.q.numel():] == 7.0).all()
    return out[at:at + b.q.numel()].view_as(b.q)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (16, 4, 128), (4, 2, 256)])
@pytest.mark.parametrize("tokens,pairs,max_q_len", [(512, 32, 0), (20, 200, 20), (8, 50, 1)])
def test_starts_that_go_back(bits, heads, kv_heads, dim, tokens, pairs, max_q_len):
    """0, T, 0, T, ..: every second sequence takes all the tokens."""
    from robustgemq_b200 import _lib
    from robustgemq_b200.serving import paged_attention

    b = Batch([(tokens, tokens + 100)], heads, kv_heads, dim, 16, bits, H16)
    want = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts, max_q_len=max_q_len)
    starts = torch.tensor([0, tokens] * pairs, dtype=torch.int32, device="cuda")
    seqs = 2 * pairs - 1
    guarded_call(b, starts, b.kv_lens.expand(seqs).contiguous(), b.page_table.expand(seqs, -1).contiguous(), max_q_len)
    assert _lib.device_error() == BAD_POSITION
    # the next call is as ever
    assert torch.equal(guarded_call(b, b.q_starts, b.kv_lens, b.page_table, max_q_len), want)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("starts", [[-5, 3, 300], [0, 1 << 30, 300], [0, -(1 << 31), 300], [300, 200, 100], [400, 500, 600]])
def test_starts_outside_the_tokens(bits, starts):
    from robustgemq_b200 import _lib

    b = Batch([(200, 300), (100, 150)], 8, 2, 64, 16, bits, B16)
    starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
    guarded_call(b, starts, b.kv_lens, b.page_table)
    assert _lib.device_error() == BAD_POSITION


@pytest.mark.parametrize("lens", [[(1 << 31) - 1, 150], [-7, 150], [-(1 << 31), 1 << 30]])
@pytest.mark.parametrize("max_q_len", [0, 1])
def test_lengths_outside_the_table(lens, max_q_len):
    from robustgemq_b200 import _lib

    b = Batch([(200, 300), (100, 150)], 8, 2, 64, 16, 8, B16)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    guarded_call(b, b.q_starts, lens, b.page_table, max_q_len)
    assert _lib.device_error() == BAD_POSITION


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("n,length", [(1, 70), (6, 3), (6, 700), (200, 70), (200, 1), (300, 700)])
@pytest.mark.parametrize("dim", [64, 256])
def test_the_widest_windows_hide_nothing(bits, n, length, dim):
    """2^31 - 1 as "no limit", also with more new tokens than positions."""
    from robustgemq_b200.serving import paged_attention

    b = Batch([(n, length), (2, 50)], 4, 2, dim, 16, bits, H16)
    want, _ = b.check()
    for window in ((1 << 31) - 1, (1 << 31) - 2, max(n, length, 50)):
        got = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts, window=window)
        assert torch.equal(got, want)


@pytest.mark.parametrize("n", [1, 40])
def test_as_many_positions_as_32_bits_take(n):
    """2^31 - 1024 positions on one page again and again, all of one weight; longer lengths
    are clamped to that and recorded. Sums in fp32 of up to 2^21 terms each, rounded or
    truncated: a quarter at most."""
    from robustgemq_b200 import _lib
    from robustgemq_b200.serving import PagedKVCache, paged_attention

    cache = PagedKVCache(1, 16, 1, 16)
    v = torch.arange(1, 17, device="cuda").half().expand(16, 1, 16).contiguous()
    cache.write(torch.zeros_like(v), v, torch.arange(16, device="cuda"))
    table = torch.zeros((1, (1 << 27) - 1), dtype=torch.int32, device="cuda")
    q = torch.randn((n, 1, 16), device="cuda").half()
    most = (1 << 31) - 1024
    for length, code in ((most, 0), (most + 1008, BAD_POSITION)):
        lens = torch.tensor([length], dtype=torch.int32, device="cuda")
        out, lse = paged_attention(q, cache, table, lens, return_lse=True)
        assert _lib.device_error() == code
        assert ((out.float() / v[0].float() - 1).abs() <= 0.25).all()
        assert ((lse - 21.4876).abs() <= 0.25).all()  # ln(2^31)
