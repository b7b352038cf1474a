"""The serving operators on B200 against their definitions in 64 bits: the paged cache
(written, read back), attention over it and the verification of drafted tokens.

Bounds are derived in ``serving_helpers`` from the operations' roundings."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from serving_helpers import ROUND, Batch, make_cache, stored_values, verify_plain

pytestmark = pytest.mark.gpu
H16, B16 = torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    from robustgemq_b200 import _lib

    _lib.device_error()
    yield
    assert _lib.device_error() == 0


# ------------------------------------------------------------------ cache
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype", [H16, B16])
@pytest.mark.parametrize("heads,dim,page,tokens,layout", [
    (1, 16, 1, 1, "own"), (3, 48, 16, 77, "pool"), (4, 128, 64, 1000, "own"), (2, 80, 32, 333, "tokens_first"),
    (5, 256, 8, 61, "pool"), (16, 64, 128, 513, "own"),
])
def test_cache_write_then_read(bits, dtype, heads, dim, page, tokens, layout):
    g = torch.Generator(device="cuda").manual_seed(tokens + bits)
    pages = -(-tokens // page) + 2
    cache = make_cache(pages, page, heads, dim, bits, dtype, layout)
    before = cache.k.clone()
    # k from a fused projection (its rows lie apart), v contiguous
    wide = torch.randn((tokens, 2 * heads * dim), generator=g, device="cuda").to(dtype)
    k = wide[:, heads * dim:].view(tokens, heads, dim)
    v = (torch.randn((tokens, heads, dim), generator=g, device="cuda") * 3).to(dtype)
    k[0, 0] = 0.0  # a row without range
    v[0, 0] = 2.5
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    cache.write(k, v, slots)
    got = cache.read(slots)
    for t, x in zip(got, (k, v)):
        assert t.dtype == dtype and t.shape == x.shape
        want = torch.from_numpy(stored_values(x.float().cpu().numpy(), bits)).to(torch.float32).to(dtype).cuda()
        assert torch.equal(t, want)
    # no other slot changed
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    same = cache.k.transpose(1, 2).reshape(pages * page, -1), before.transpose(1, 2).reshape(pages * page, -1)
    a, b = (x[rest] for x in same)
    assert torch.equal(a.view(torch.int16) if bits == 16 else a, b.view(torch.int16) if bits == 16 else b)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_cache_negative_slots_and_empty_calls(bits):
    cache = make_cache(4, 16, 2, 64, bits, H16)
    x = torch.randn((3, 2, 64), device="cuda").half()
    slots = torch.tensor([-1, 5, -7], device="cuda")
    cache.write(x, x, slots)
    k, v = cache.read(slots)
    assert (k[0] == 0).all() and (v[2] == 0).all() and torch.isfinite(k).all()
    cache.write(x[:0], x[:0], slots[:0])
    k, _ = cache.read(slots[:0])
    assert k.shape == (0, 2, 64)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_cache_poisoned_row_stays_alone(bits, value):
    cache = make_cache(2, 16, 3, 64, bits, B16)
    x = torch.randn((4, 3, 64), device="cuda").to(B16)
    bad = x.clone()
    bad[2, 1, 63] = value
    slots = torch.arange(4, device="cuda")
    cache.write(bad, x, slots)
    k, v = cache.read(slots)
    assert torch.isnan(k[2, 1]).all()
    k[2, 1] = 0
    assert torch.isfinite(k).all() and torch.isfinite(v).all()


def test_cache_slot_past_the_end_is_recorded():
    from robustgemq_b200 import _lib

    cache = make_cache(2, 16, 1, 64, 16, H16)
    x = torch.ones((2, 1, 64), device="cuda").half()
    cache.write(x, x, torch.tensor([32, 31], device="cuda"))
    assert _lib.device_error() == 10
    k, _ = cache.read(torch.tensor([31, 1 << 40], device="cuda"))
    assert (k[0] == 1).all() and (k[1] == 0).all()
    assert _lib.device_error() == 10


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("dtype", [H16, B16])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 128, 16), (8, 1, 64, 64), (6, 2, 80, 32), (3, 1, 256, 8)])
@pytest.mark.parametrize("lens", [
    [(1, 1)], [(1, 63), (1, 64), (1, 65), (1, 1000)], [(5, 5), (2, 300), (9, 129)],
    [(40, 40), (1, 700), (0, 30), (130, 517)],
], ids=["one", "decode", "drafts", "mixed"])
def test_attention(bits, dtype, heads, kv_heads, dim, page, lens):
    Batch(lens, heads, kv_heads, dim, page, bits, dtype, seed=dim + bits).check(
        max_q_len=max(n for n, _ in lens), max_kv_len=max(n for _, n in lens))


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("window", [1, 7, 128, 400])
@pytest.mark.parametrize("lens", [[(1, 900), (3, 40)], [(257, 600), (1, 5)]], ids=["few", "many"])
def test_attention_window(bits, window, lens):
    Batch(lens, 8, 2, 128, 32, bits, H16, seed=window).check(window=window)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("q_len", [1, 3, 200])
def test_attention_rows_that_see_nothing(bits, q_len):
    """More new tokens than positions: the first ones lie before position 0."""
    b = Batch([(q_len, 1), (q_len, 0), (q_len, max(1, q_len - 1)), (q_len, 70)], 4, 2, 64, 16, bits, H16)
    out, lse = b.check()
    assert (out[q_len:2 * q_len] == 0).all() and (lse[q_len:2 * q_len] == -math.inf).all()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("layout", ["pool", "tokens_first"])
def test_attention_strided_cache_and_queries(bits, layout):
    b = Batch([(1, 333), (70, 200)], 8, 4, 128, 16, bits, B16, layout=layout)
    wide = torch.zeros((b.tokens, 3, 8, 128), dtype=B16, device="cuda")
    wide[:, 1] = b.q
    b.q = wide[:, 1]
    b.page_table = torch.cat([b.page_table, b.page_table], 1)[:, :b.page_table.shape[1]]
    b.check()
    b.q = b.q.transpose(0, 1).contiguous().transpose(0, 1)  # heads first in memory
    b.check()


@pytest.mark.parametrize("bits,dtype", [(16, H16), (16, B16), (8, H16), (4, B16)])
def test_attention_equal_chunks_without_starts(bits, dtype):
    Batch([(4, 100), (4, 31), (4, 4)], 4, 4, 64, 16, bits, dtype).check(use_starts=False)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("lens", [[(1, 20000)], [(1, 9000), (1, 17), (2, 4097)], [(150, 5000)], [(300, 2500), (64, 7000)]],
                         ids=["long", "uneven", "chunk", "chunks"])
def test_attention_long_axis_is_split_and_joined(bits, lens):
    Batch(lens, 8, 2, 128, 64, bits, H16, seed=5).check(max_q_len=max(n for n, _ in lens),
                                                        max_kv_len=max(n for _, n in lens))


@pytest.mark.parametrize("max_q_len,max_kv_len", [(1, 1), (2, 64), (1000, 1), (0, 0)])
def test_attention_wrong_bounds_cost_time_only(max_q_len, max_kv_len):
    Batch([(33, 300), (1, 2000), (260, 400)], 4, 2, 64, 16, 16, H16).check(max_q_len=max_q_len, max_kv_len=max_kv_len)


@pytest.mark.parametrize("gain", [30.0, 0.0])
@pytest.mark.parametrize("q_len", [1, 140])
def test_attention_sharp_and_flat_scores(gain, q_len):
    """Scores of some hundreds (one key takes all) and scores of zero."""
    Batch([(q_len, 1500)], 4, 1, 128, 32, 16, H16, q_gain=gain).check()
    Batch([(q_len, 1500)], 4, 1, 128, 32, 8, B16, q_gain=gain).check()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("n,length", [(1, 300), (9, 700), (200, 600)])
def test_attention_steps_of_every_size(bits, n, length):
    """Rows of equal values (a step of 2^-64, all of the value in the base), zero rows, and
    steps that differ by 2^20 between positions, larger ones later."""
    b = Batch([(n, length)], 4, 2, 64, 16, bits, H16, seed=n)
    g = torch.Generator(device="cuda").manual_seed(7)
    k = torch.randn((length, 2, 64), generator=g, device="cuda").half()
    v = torch.randn((length, 2, 64), generator=g, device="cuda").half()
    v[::3] = torch.randn((v[::3].shape[0], 2, 1), generator=g, device="cuda").half()
    v[1::7] = 0.0
    k[5::9] = 0.0
    k[7::11] = 0.25
    v[length // 2:] *= 2.0 ** 10
    v[:length // 4] *= 2.0 ** -10
    b.put(0, torch.arange(length, device="cuda"), k, v)
    b.k[0] = torch.from_numpy(stored_values(k.float().cpu().numpy(), bits)).cuda()
    b.v[0] = torch.from_numpy(stored_values(v.float().cpu().numpy(), bits)).cuda()
    b.check()
    # nothing but rows of equal values
    v = torch.randn((length, 2, 1), generator=g, device="cuda").half().expand(length, 2, 64).contiguous()
    b.put(0, torch.arange(length, device="cuda"), k, v)
    b.v[0] = torch.from_numpy(stored_values(v.float().cpu().numpy(), bits)).cuda()
    b.check()


@pytest.mark.parametrize("n", [1, 40, 150])
@pytest.mark.parametrize("bits", [16, 4])
def test_attention_negative_scale(n, bits):
    Batch([(n, 400)], 4, 2, 64, 16, bits, B16).check(scale=-0.2)
    Batch([(n, 400)], 4, 2, 64, 16, bits, H16).check(scale=0.0)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("n,length,hit", [(1, 300, 100), (6, 300, 297), (6, 300, 100), (200, 500, 400), (200, 500, 350)])
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_attention_non_finite_rows_reach_only_who_sees_them(bits, n, length, hit, which, value):
    """A key or value with a NaN or an infinity at one position: the rows before it are
    what they are without it, the rows that see it are not finite (an infinite key may
    also just take, or lose, all the weight)."""
    from robustgemq_b200.serving import paged_attention

    b = Batch([(n, length), (n, 64)], 4, 2, 64, 16, bits, H16, seed=hit)
    ref, ref_lse = b.check()
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn((1, 2, 64), generator=g, device="cuda").half()
    v = torch.randn((1, 2, 64), generator=g, device="cuda").half()
    if which != "v":
        k[0, 0, 5] = value
    if which != "k":
        v[0, 0, 9] = value
    b.put(0, torch.tensor([hit], device="cuda"), k, v)
    out, lse = paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=b.q_starts, return_lse=True)
    first = max(0, hit - (length - n))  # the first row that sees the position
    u = ROUND[H16]
    assert torch.isfinite(out[:first]).all()
    # the rows before it: the same up to the split's own roundings
    assert ((out[:first].float() - ref[:first].float()).abs() <= 4 * u * (1 + ref[:first].float().abs())).all()
    assert torch.isfinite(out[n:]).all() and torch.equal(lse[n:], ref_lse[n:])
    seers = out[first:n, :2]  # query heads of KV head 0
    if which != "k":
        column = seers[..., 9] if bits == 16 else seers
        if value != value or bits != 16:
            assert torch.isnan(column).all() if which == "v" else not torch.isfinite(column).all()
    elif value != value or bits != 16:
        assert torch.isnan(seers).all()
    assert torch.isfinite(out[first:n, 2:]).all()


def test_attention_cache_past_32_bit_offsets():
    """Pages whose byte offset passes 2^32: a cache of 4.5 GiB a side, sequences on its
    last pages."""
    from robustgemq_b200.serving import PagedKVCache, paged_attention

    page, heads, dim = 64, 4, 128
    pages = (9 << 29) // (page * heads * dim * 2)
    cache = PagedKVCache(pages, page, heads, dim)
    g = torch.Generator(device="cuda").manual_seed(0)
    for n in (1, 130):
        length = 200
        k = torch.randn((length, heads, dim), generator=g, device="cuda").half()
        v = torch.randn((length, heads, dim), generator=g, device="cuda").half()
        table = torch.arange(pages - 4, pages, device="cuda", dtype=torch.int32)[None]
        slots = (pages - 4) * page + torch.arange(length, device="cuda")
        cache.write(k, v, slots)
        assert torch.equal(cache.read(slots)[0], k)
        q = torch.randn((n, heads, dim), generator=g, device="cuda").half()
        lens = torch.tensor([length], dtype=torch.int32, device="cuda")
        got = paged_attention(q, cache, table, lens)
        small = PagedKVCache(4, page, heads, dim)
        small.write(k, v, torch.arange(length, device="cuda"))
        want = paged_attention(q, small, table - (pages - 4), lens)
        assert torch.equal(got, want)


def test_attention_bad_lengths_and_pages_are_recorded():
    from robustgemq_b200 import _lib
    from robustgemq_b200.serving import paged_attention

    for n in (1, 140):
        b = Batch([(n, 100)], 2, 2, 64, 16, 16, H16)
        want = paged_attention(b.q, b.cache, b.page_table, b.kv_lens)
        torch.cuda.synchronize()
        assert _lib.device_error() == 0
        cap = b.page_table.shape[1] * 16
        paged_attention(b.q, b.cache, b.page_table, torch.full_like(b.kv_lens, cap + 1))
        assert _lib.device_error() == 10
        table = b.page_table.clone()
        table[0, 2] = -1
        paged_attention(b.q, b.cache, table, b.kv_lens)
        assert _lib.device_error() == 10
        paged_attention(b.q, b.cache, b.page_table, b.kv_lens, q_starts=torch.tensor([0, n + 5], dtype=torch.int32, device="cuda"))
        assert _lib.device_error() == 10
        assert torch.equal(paged_attention(b.q, b.cache, b.page_table, b.kv_lens), want)


def test_attention_leaves_tokens_outside_every_sequence():
    from robustgemq_b200 import _lib

    b = Batch([(1, 40), (3, 50)], 2, 1, 64, 16, 16, H16)
    lib = _lib.load()
    q = torch.cat([b.q, b.q])  # four tokens of padding
    out = torch.full_like(q, 7.0)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    _lib.check(lib.gemq_paged_attention(
        ctypes.cast(b.cache.c_struct, ctypes.POINTER(_lib.KvCacheT)), q.data_ptr(), q.stride(0), 8, 2, b.page_table.data_ptr(), b.page_table.stride(0),
        b.page_table.shape[1], b.kv_lens.data_ptr(), b.q_starts.data_ptr(), 2, 3, 50, 0.125, 0, out.data_ptr(), None,
        ws.data_ptr(), ws.numel(), _lib.stream_ptr(q.device)))
    o, _, tol, _ = b.expect(0.125)
    assert ((out[:4].double() - o).abs() <= tol).all()
    assert (out[4:] == 7.0).all()


def test_attention_same_bits_every_time():
    """The joined parts are summed in a fixed order."""
    b = Batch([(1, 3000), (2, 5000), (1, 10)], 8, 2, 128, 16, 8, H16)
    first, lse = b.check()
    for _ in range(5):
        out, again = b.check()
        assert torch.equal(out, first) and torch.equal(again, lse)


def test_step_on_another_stream_and_in_a_graph():
    """Write and attention captured once and replayed with new contents, on a stream of
    the caller's."""
    from robustgemq_b200.serving import paged_attention

    b = Batch([(1, 200), (1, 77)], 4, 2, 64, 16, 8, H16)
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn((2, 2, 64), generator=g, device="cuda").half() for _ in range(2))
    slots = torch.stack([b.slots(0, torch.tensor(199, device="cuda")), b.slots(1, torch.tensor(76, device="cuda"))])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.cache.write(k, v, slots)
        eager = paged_attention(b.q, b.cache, b.page_table, b.kv_lens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            b.cache.write(k, v, slots)
            out = paged_attention(b.q, b.cache, b.page_table, b.kv_lens)
        for i in range(3):
            k.copy_(torch.randn((2, 2, 64), generator=g, device="cuda"))
            graph.replay()
            s.synchronize()
            replayed = out.clone()
            b.cache.write(k, v, slots)
            assert torch.equal(replayed, paged_attention(b.q, b.cache, b.page_table, b.kv_lens))
            assert not torch.equal(replayed, eager)
    torch.cuda.current_stream().wait_stream(s)


# ------------------------------------------------------------------ verification
def _verify_inputs(B, n, V, dtype, seed, probs=None, agree=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn((B, n + 1, V), generator=g, device="cuda") * 3
    draft = torch.softmax(logits[:, :n] + torch.randn((B, n, V), generator=g, device="cuda") * agree, -1)
    race = torch.empty((B, n, V), device="cuda").exponential_(generator=g)
    x = (draft / race).argmax(-1) if probs is not None else draft.argmax(-1)
    u = torch.rand((B, n), generator=g, device="cuda")
    e = torch.empty((B, V), device="cuda").exponential_(generator=g)
    return logits.to(dtype), x, u, e, None if probs is None else draft.to(probs)


def _check_verify(logits, x, u, e, probs=None, lens=None, temps=None):
    from robustgemq_b200.serving import verify_draft

    r = verify_draft(logits, x, u, e, draft_probs=probs, draft_lens=lens, temperature=temps)
    host = [None if t is None else (t.float() if t.is_floating_point() else t).cpu().numpy()
            for t in (logits, x, u, e, probs, lens, temps)]
    tokens, accepted, lp, margin = verify_plain(*host)
    sure = margin > 1e-4  # fp32 logits / T and exp are good to about 1e-5
    assert sure.mean() > 0.8
    assert np.array_equal(r.tokens.cpu().numpy()[sure], tokens[sure])
    assert np.array_equal(r.num_accepted.cpu().numpy()[sure], accepted[sure])
    # logits of some tens over T >= 0.3 rounded to fp32, a sum in fp32: 1e-5 is 5 times that
    assert np.abs(r.logprobs.cpu().numpy()[sure] - lp[sure]).max() <= 1e-5 * (1 + np.abs(lp).max())
    return r


@pytest.mark.parametrize("dtype", [H16, B16, torch.float32])
@pytest.mark.parametrize("probs", [None, torch.float32, H16, B16])
@pytest.mark.parametrize("B,n,V", [(1, 1, 1), (3, 1, 7), (5, 4, 1003), (16, 7, 32001), (2, 40, 513), (70, 3, 4096)])
def test_verify(dtype, probs, B, n, V):
    _check_verify(*_verify_inputs(B, n, V, dtype, B + V, probs))


@pytest.mark.parametrize("probs", [None, torch.float32])
def test_verify_lengths_and_temperatures(probs):
    B, n, V = 30, 5, 2001
    logits, x, u, e, q = _verify_inputs(B, n, V, torch.float32, 3, probs)
    lens = (torch.arange(B, device="cuda") % (n + 1)).int()
    temps = torch.rand(B, device="cuda") + 0.3
    temps[::3] = 0.0
    r = _check_verify(logits, x, u, e, q, lens, temps)
    assert (r.num_accepted <= lens).all()
    greedy = logits.argmax(-1)
    for b in range(0, B, 3):
        a = int(r.num_accepted[b])
        assert torch.equal(r.tokens[b, :a + 1], greedy[b, :a + 1])


def test_verify_strided_logits():
    logits, x, u, e, q = _verify_inputs(4, 3, 1001, H16, 11, torch.float32)
    wide = torch.zeros((4, 6, 1003), dtype=H16, device="cuda")
    wide[:, 1:5, 1:1002] = logits
    a = _check_verify(wide[:, 1:5, 1:1002], x, u, e, q)
    b = _check_verify(logits, x, u, e, q)
    assert torch.equal(a.tokens, b.tokens)
    c = _check_verify(logits.transpose(1, 2).contiguous().transpose(1, 2), x, u, e, q)
    assert torch.equal(c.tokens, b.tokens)


def test_verify_masked_vocabulary_and_rows_without_distribution():
    B, n, V = 8, 2, 500
    logits, x, u, e, _ = _verify_inputs(B, n, V, torch.float32, 21)
    lowest = torch.finfo(torch.float32).min
    logits[0, :, 100:] = -math.inf       # masked, few left
    logits[1, :, 1:] = lowest            # the type's lowest value: no weight
    x[1] = 0
    logits[2, 1] = -math.inf             # nothing left
    logits[3, 0, 7] = math.nan
    logits[4, 2, 499] = math.inf
    logits[5] = -math.inf
    logits[5, :, 499] = 0.0              # one token left
    x[6, 0], x[7, 1] = -5, V             # drafts that are no tokens
    u[2, 0] = u[4] = 0.0
    r = _check_verify(logits, x, u, e)
    t = r.tokens.cpu()
    assert int(t[3, 0]) == -1 and int(r.num_accepted[3]) == 0
    assert t[2, 1] == -1 or int(r.num_accepted[2]) < 1
    assert int(t[5, int(r.num_accepted[5])]) == 499
    assert int(r.num_accepted[6]) == 0 and int(t[6, 0]) >= 0
    assert int(r.num_accepted[7]) <= 1
    temps = torch.tensor([1.0, -1.0, math.nan] + [0.0] * 5, device="cuda")
    r = _check_verify(logits, x, u, e, temps=temps)
    assert int(r.tokens[1, 0]) == -1 and int(r.tokens[2, 0]) == -1


def test_verify_draft_equal_to_the_target_takes_everything():
    """q = p: u q < p for every u below 1 up to the last bits, and where the difference
    leaves nothing the token comes from p."""
    B, n, V = 64, 4, 300
    g = torch.Generator(device="cuda").manual_seed(2)
    logits = torch.randn((B, n + 1, V), generator=g, device="cuda")
    probs = torch.softmax(logits, -1)[:, :n].contiguous()
    x = torch.randint(0, V, (B, n), generator=g, device="cuda")
    u = torch.rand((B, n), generator=g, device="cuda") * 0.999
    e = torch.empty((B, V), device="cuda").exponential_(generator=g)
    from robustgemq_b200.serving import verify_draft

    r = verify_draft(logits, x, u, e, draft_probs=probs)
    assert (r.num_accepted == n).all()
    # certain rejection (u q = inf) of a draft whose p - q is nowhere above zero
    big = verify_draft(logits, x, torch.full_like(u, math.inf), e, draft_probs=probs * 2)
    assert (big.num_accepted == 0).all()
    want = (torch.softmax(logits[:, 0].double(), -1) / e.double()).argmax(-1)
    assert torch.equal(big.tokens[:, 0], want)


def test_verify_ties_go_to_the_lowest_index():
    from robustgemq_b200.serving import verify_draft

    V = 9000
    logits = torch.zeros((1, 2, V), device="cuda")
    noise = torch.ones((1, V), device="cuda")
    u = torch.zeros((1, 1), device="cuda")
    r = verify_draft(logits, torch.zeros((1, 1), dtype=torch.int64, device="cuda"), u, noise)
    assert r.tokens.tolist() == [[0, 0]]
    r = verify_draft(logits, torch.zeros((1, 1), dtype=torch.int64, device="cuda"), u + 0.9, noise)
    assert r.tokens.tolist() == [[1, -1]]
    r = verify_draft(logits, torch.full((1, 1), 5, device="cuda"), u, noise, temperature=torch.zeros(1, device="cuda"))
    assert r.tokens.tolist() == [[0, -1]]


@pytest.mark.parametrize("sampled", [True, False])
def test_verify_keeps_the_targets_distribution(sampled):
    """The first token's distribution over 65,535 sequences that share p and q is p: each
    frequency within 5 standard deviations."""
    from robustgemq_b200.serving import verify_draft

    B, V = 65535, 12
    g = torch.Generator(device="cuda").manual_seed(4)
    p = torch.softmax(torch.randn(V, generator=g, device="cuda") * 1.5, -1)
    q = torch.softmax(torch.randn(V, generator=g, device="cuda") * 1.5, -1)
    logits = p.log().expand(B, 2, V).contiguous()
    if sampled:
        x = torch.multinomial(q, B, replacement=True, generator=g).view(B, 1)
        probs = q.expand(B, 1, V).contiguous()
    else:
        x, probs = torch.full((B, 1), 3, device="cuda"), None
    u = torch.rand((B, 1), generator=g, device="cuda")
    e = torch.empty((B, V), device="cuda").exponential_(generator=g)
    r = verify_draft(logits, x, u, e, draft_probs=probs)
    freq = torch.bincount(r.tokens[:, 0], minlength=V).double() / B
    assert ((freq - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / B).sqrt()).all()


def test_verify_vocabulary_of_one_part_or_many_gives_the_same():
    """The race is a maximum: adding tokens without weight, hence other parts, changes
    nothing."""
    from robustgemq_b200.serving import verify_draft

    logits, x, u, e, q = _verify_inputs(3, 2, 1500, torch.float32, 8, torch.float32)
    a = verify_draft(logits, x, u, e, draft_probs=q)
    pad = 150000 - 1500
    b = verify_draft(torch.nn.functional.pad(logits, (0, pad), value=-math.inf), x, u,
                     torch.nn.functional.pad(e, (0, pad), value=1e-30), draft_probs=torch.nn.functional.pad(q, (0, pad)))
    assert torch.equal(a.tokens, b.tokens) and torch.equal(a.num_accepted, b.num_accepted)
