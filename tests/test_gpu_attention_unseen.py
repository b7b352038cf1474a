"""Large finite values that a row does not see, or that have no weight in it, against the
definition in 64 bits with a bound a row: nothing in it is taken over keys that the row
does not see.

Bound of a row's output, beyond what ``serving_helpers`` derives for scores and sums: a
weight is rounded to 16 bits, by its roundoff u relatively or, where fp16 runs out of
exponent, by 2^-25 of the row's largest and by no more than itself. With codes the
rounded weight is the one times the value's step, so "largest" is that of weight times
step, and the error counts in steps times codes: no more than 1.1 of the largest value of
that key (codes of 4 bits reach 8/15 of the range from their middle)."""

from __future__ import annotations

import math

import pytest
import torch

from serving_helpers import ROUND, Batch, stored_values

pytestmark = pytest.mark.gpu
H16, B16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    from robustgemq_b200 import _lib

    _lib.device_error()
    yield
    assert _lib.device_error() == 0


def check_rows(b, seq, window=0):
    """Every row of sequence ``seq`` of the batch by its own bound."""
    from robustgemq_b200.serving import paged_attention

    scale = b.dim ** -0.5
    got, lse = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts, scale=scale, window=window,
                               return_lse=True)
    at = sum(n for n, _ in b.lens[:seq])
    n, length = b.lens[seq]
    q = b.q[at:at + n].double()
    g = b.heads // b.kv_heads
    k, v = b.k[seq].repeat_interleave(g, 1), b.v[seq].repeat_interleave(g, 1)
    pos = torch.arange(length - n, length, device="cuda")[:, None]
    key = torch.arange(length, device="cuda")[None]
    seen = (key <= pos) & ((key > pos - window) if window else (key >= 0))  # [q, k]
    u = ROUND[b.dtype]
    for h in range(b.heads):
        s = (q[:, h] @ k[:, h].T) * scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        row = torch.logsumexp(s, -1)
        p = torch.exp(s - row[:, None])
        o = p @ v[:, h]
        a = p @ v[:, h].abs()
        mag = torch.where(seen, (q[:, h].abs() @ k[:, h].abs().T) * scale, torch.zeros_like(s)).amax(-1)
        top = torch.where(seen, s.abs(), torch.zeros_like(s)).amax(-1)
        # the dot product of D terms in fp32; scores and log2 of the step (64 at most) as
        # fp32 powers of two
        rel = 2 * mag * b.dim * 2.0 ** -23 + (1.45 * top + 64) * 2.0 ** -22 + length * 2.0 ** -23
        size = v[:, h].abs().amax(-1)
        unit = torch.ones_like(size) if b.bits == 16 else size
        w = p * unit
        lost = torch.minimum(w, 2.0 ** -25 * w.amax(-1, keepdim=True))
        tiny = lost @ (size if b.bits == 16 else torch.full_like(size, 1.1))
        tol = u * (o.abs() + a) * 1.01 + rel[:, None] * a + tiny[:, None] + 2.0 ** -24
        off = (got[at:at + n, h].double() - o).abs()
        bad = ~(off <= tol)
        assert not bad.any(), (f"head {h}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, "
                               f"worst {float((off / tol).nan_to_num(1e9).max()):.3g} times the bound")
        assert ((lse[at:at + n, h].double() - row).abs() <= rel + 2.0 ** -20 * (1 + row.abs())).all()


def replace(b, seq, positions, k, v):
    b.put(seq, positions, k, v)
    b.k[seq][positions] = torch.from_numpy(stored_values(k.float().cpu().numpy(), b.bits)).cuda()
    b.v[seq][positions] = torch.from_numpy(stored_values(v.float().cpu().numpy(), b.bits)).cuda()


def make(n, length, heads, kv_heads, dim, bits, dtype, loud, gain, k_of=None):
    """A sequence whose values are of 0.01, those at the positions ``loud`` times ``gain``."""
    b = Batch([(n, length), (3, 40)], heads, kv_heads, dim, 16, bits, dtype, seed=dim + n)
    gen = torch.Generator(device="cuda").manual_seed(n)
    at = torch.arange(length, device="cuda")
    k = torch.randn((length, kv_heads, dim), generator=gen, device="cuda")
    v = torch.randn((length, kv_heads, dim), generator=gen, device="cuda") * 0.01
    v[loud] *= gain
    if k_of is not None:
        k_of(k)
    replace(b, 0, at, k.to(dtype), v.to(dtype))
    return b


GAIN = {H16: 2.0 ** 20, B16: 2.0 ** 40}  # fp16 values of some 10^4
SHAPES = [(4, 2, 64), (8, 1, 128), (3, 1, 80), (4, 4, 256)]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype", [H16, B16])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("n,length", [(3, 200), (60, 400), (300, 700)])
def test_loud_values_after_a_row(bits, dtype, heads, kv_heads, dim, n, length):
    """In the chunk's last third: in the diagonal tile of some rows, in later ones of others."""
    b = make(n, length, heads, kv_heads, dim, bits, dtype, torch.arange(length - (n + 2) // 3, length, 7), GAIN[dtype])
    check_rows(b, 0)
    check_rows(b, 1)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype", [H16, B16])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("n,length", [(3, 200), (60, 400), (300, 700)])
def test_loud_values_left_of_the_window(bits, dtype, heads, kv_heads, dim, n, length):
    """Just before the first row's window (which no row sees) and inside it (which the
    first rows see and the others do not)."""
    window = 50
    first = length - n - window
    b = make(n, length, heads, kv_heads, dim, bits, dtype, torch.tensor([first - 9, first, first + 1, first + 20]), GAIN[dtype])
    check_rows(b, 0, window)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype", [H16, B16])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("n,length", [(3, 200), (60, 400), (300, 700)])
def test_loud_values_without_weight(bits, dtype, heads, kv_heads, dim, n, length):
    """Keys that every row sees with scores some 80 below the others, so that even their
    loud values come to nothing."""
    loud = torch.tensor([5, 33, 120])

    def k_of(k):
        k[..., 0] = 0.0
        k[loud, :, 0] = -20.0 * dim ** 0.5

    b = make(n, length, heads, kv_heads, dim, bits, dtype, loud, GAIN[H16], k_of)
    b.q[..., 0] = 4.0
    check_rows(b, 0)


def large_equal(bits, heads, kv_heads, dim, n, length, size):
    """A batch, its keys and bf16 value rows of one large value each."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    b = Batch([(n, length), (3, 40)], heads, kv_heads, dim, 16, bits, B16, seed=dim + n)
    k = torch.randn((length, kv_heads, dim), generator=gen, device="cuda").to(B16)
    v = (torch.rand((length, kv_heads, 1), generator=gen, device="cuda") * 2 - 1) * size
    return b, k, v.expand(length, kv_heads, dim).to(B16).contiguous()


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("n,length", [(3, 200), (60, 400), (300, 700)])
@pytest.mark.parametrize("size", [1e12, 1e20, 1e30, 1e38])
def test_rows_of_large_equal_values_at_4_bits(heads, kv_heads, dim, n, length, size):
    """Rows whose step is 2^-64, with all of the value in the base: alone, and between rows of
    zeros."""
    b, k, v = large_equal(4, heads, kv_heads, dim, n, length, size)
    at = torch.arange(length, device="cuda")
    replace(b, 0, at, k, v)
    check_rows(b, 0)
    v[::2] = 0.0
    replace(b, 0, at, k, v)
    check_rows(b, 0)


@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("n,length", [(3, 200), (60, 400), (300, 700)])
@pytest.mark.parametrize("size", [1e12, 1e20, 1e30, 1e38])
def test_rows_of_large_equal_values_at_8_bits(heads, kv_heads, dim, n, length, size):
    """Between rows of zeros, whose step is 2^-64: the rows of zeros keep their weight, or,
    where the steps lie too far apart for that, every row that sees a large value is NaN."""
    from robustgemq_b200.serving import paged_attention

    b, k, v = large_equal(8, heads, kv_heads, dim, n, length, size)
    v = (v.float() / 127).to(B16)  # 127 times the largest has to stay in fp32
    at = torch.arange(length, device="cuda")
    v[::2] = 0.0
    replace(b, 0, at, k, v)
    if size / 127 / 127 < 2.0 ** 38:
        check_rows(b, 0)
    else:
        out = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts)
        assert torch.isnan(out[:n]).all()
        check_rows(b, 1)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("n,length", [(3, 200), (60, 400), (300, 700)])
def test_steps_that_are_none_stay_with_the_rows_that_see_them(bits, heads, kv_heads, dim, n, length):
    """A value row of 1e30 in the chunk: NaN from its position on, nothing before it."""
    from robustgemq_b200.serving import paged_attention

    loud = length - (n + 2) // 3
    b = make(n, length, heads, kv_heads, dim, bits, B16, torch.tensor([], dtype=torch.int64), 1.0)
    want = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts)
    v = torch.randn((1, kv_heads, dim), device="cuda").mul_(1e30).to(B16)
    b.put(0, torch.tensor([loud], device="cuda"), torch.zeros_like(v), v)
    out = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts)
    first = loud - (length - n)
    assert torch.equal(out[:first], want[:first]) and torch.equal(out[n:], want[n:])
    assert torch.isnan(out[first:n]).all()
