"""Attention of chunks over a paged cache with heads of more than 128 columns, against its
definition in 64 bits (bounds as in ``serving_helpers``)."""

from __future__ import annotations

import math

import pytest
import torch

from serving_helpers import ROUND, Batch

pytestmark = pytest.mark.gpu
H16, B16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    from robustgemq_b200 import _lib

    _lib.device_error()
    yield
    assert _lib.device_error() == 0


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype", [H16, B16])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 256, 16), (6, 2, 144, 32), (8, 1, 192, 128), (3, 1, 240, 8)])
@pytest.mark.parametrize("lens", [[(33, 33)], [(40, 700), (1, 64), (0, 30), (130, 517)], [(129, 65), (300, 1000)]],
                         ids=["start", "mixed", "before"])
def test_wide_heads(bits, dtype, heads, kv_heads, dim, page, lens):
    Batch(lens, heads, kv_heads, dim, page, bits, dtype, seed=dim + bits).check(
        max_q_len=max(n for n, _ in lens), max_kv_len=max(n for _, n in lens))


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("window", [1, 63, 400])
def test_wide_heads_window(bits, window):
    Batch([(257, 900), (64, 70)], 4, 2, 256, 32, bits, H16, seed=window).check(window=window)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens", [[(150, 9000)], [(300, 2500), (64, 7000)]], ids=["one", "two"])
def test_wide_heads_split_along_the_keys(bits, lens):
    Batch(lens, 4, 1, 256, 64, bits, B16, seed=5).check(max_q_len=max(n for n, _ in lens),
                                                        max_kv_len=max(n for _, n in lens))


@pytest.mark.parametrize("layout", ["pool", "tokens_first"])
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_wide_heads_strides_and_negative_scale(bits, layout):
    b = Batch([(70, 200), (40, 333)], 4, 2, 256, 16, bits, B16, layout=layout)
    b.q = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    b.check(scale=-0.1)


@pytest.mark.parametrize("bits", [16, 8])
def test_wide_heads_sharp_scores(bits):
    """Scores of some hundreds: the running reference moves often."""
    Batch([(140, 1500)], 4, 1, 256, 32, bits, H16, q_gain=20.0).check()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_wide_heads_what_is_not_seen_does_not_count(bits, value):
    """A value with a NaN or an infinity at one position, in each half of the columns: the
    rows before it are what they are without it."""
    from robustgemq_b200.serving import paged_attention

    for col in (3, 250):
        b = Batch([(150, 400)], 4, 2, 256, 16, bits, H16)
        out, _ = b.check()
        at = 300
        v = torch.zeros((1, 2, 256), device="cuda").half()
        v[0, :, col] = value
        b.put(0, torch.tensor([at], device="cuda"), torch.ones_like(v), v)
        got = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts)
        before = at - 250  # rows of positions 250 to 299
        # the same up to the split's own roundings
        bound = 4 * ROUND[H16] * (1 + out[:before].float().abs())
        assert ((got[:before].float() - out[:before].float()).abs() <= bound).all()
        assert not torch.isfinite(got[before:, :, col]).any()
