"""The serving operators' refusals, on the CPU: what the C ABI and the Python entry points
check before they touch the device."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from serving_helpers import quantise_rows, verify_plain


def _cache(**kw):
    from robustgemq_b200._lib import KvCacheT

    c = KvCacheT()
    c.k = c.v = 0x10000
    c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.bits, c.dtype = 8, 4, 16, 128, 16, 0
    c.strides = (4 * 16 * 256, 16 * 256, 256)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _status(rc):
    from robustgemq_b200 import _lib

    return rc, _lib.load().gemq_last_error_string().decode()


INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4
BAD_CACHES = [
    (dict(bits=3), INVALID, "bits"), (dict(dtype=2), INVALID, "dtype"), (dict(num_pages=0), INVALID, "size"),
    (dict(head_dim=-16), INVALID, "size"), (dict(head_dim=72), UNSUPPORTED, "head_dim"),
    (dict(head_dim=272), UNSUPPORTED, "head_dim"), (dict(page_size=24), UNSUPPORTED, "page_size"),
    (dict(num_pages=1 << 30), UNSUPPORTED, "2^31"), (dict(k=None), INVALID, "null"),
    (dict(bits=8), INVALID, "null"), (dict(k=0x10008), UNSUPPORTED, "aligned"),
    (dict(strides=(8, 256, 256)), UNSUPPORTED, "aligned"), (dict(strides=(-256, 256, 256)), UNSUPPORTED, "aligned"),
    (dict(bits=4, k_scale=0x1004, v_scale=0x1000), UNSUPPORTED, "aligned"),
]


@pytest.mark.parametrize("change,code,text", BAD_CACHES)
def test_bad_caches_are_refused_everywhere(change, code, text):
    from robustgemq_b200 import _lib

    lib = _lib.load()
    ref = ctypes.byref(_cache(**change))
    calls = [
        lib.gemq_kv_cache_write(ref, 0x1000, 0x1000, 512, 128, 512, 128, 0x1000, 4, None),
        lib.gemq_kv_cache_read(ref, 0x1000, 4, 0x1000, 0x1000, None),
        lib.gemq_paged_attention(ref, 0x1000, 512, 4, 4, 0x1000, 8, 8, 0x1000, None, 4, 0, 0, 1.0, 0, 0x1000, None,
                                 None, 0, None),
    ]
    for rc in calls:
        assert rc == code
        assert text in lib.gemq_last_error_string().decode()
    assert lib.gemq_paged_attention_workspace_size(ref, 4, 4, 4, 8, 0, 0) == 0


@pytest.mark.parametrize("args,code,text", [
    (dict(k=None), INVALID, "null"), (dict(slots=None), INVALID, "null"), (dict(tokens=-1), INVALID, "negative"),
    (dict(tokens=1 << 29), UNSUPPORTED, "2^29"), (dict(k=0x1008), UNSUPPORTED, "16-byte"),
    (dict(kts=513), UNSUPPORTED, "16-byte"),
])
def test_cache_write_refusals(args, code, text):
    from robustgemq_b200 import _lib

    a = dict(k=0x1000, slots=0x1000, tokens=4, kts=512) | args
    rc, msg = _status(_lib.load().gemq_kv_cache_write(ctypes.byref(_cache()), a["k"], 0x1000, a["kts"], 128, 512, 128,
                                                      a["slots"], a["tokens"], None))
    assert rc == code and text in msg


@pytest.mark.parametrize("args,code,text", [
    (dict(heads=6), INVALID, "multiple"), (dict(heads=0), INVALID, "size"), (dict(tokens=-1), INVALID, "size"),
    (dict(window=-1), INVALID, "window"), (dict(scale=float("nan")), INVALID, "finite"),
    (dict(scale=float("inf")), INVALID, "finite"), (dict(tokens=5), INVALID, "q_starts"), (dict(q=None), INVALID, "null"),
    (dict(lens=None), INVALID, "null"), (dict(table=None), INVALID, "null"), (dict(out=None), INVALID, "null"),
    (dict(q=0x1004), UNSUPPORTED, "16-byte"), (dict(qts=516), UNSUPPORTED, "multiple of 8"),
    (dict(pages=1 << 28), UNSUPPORTED, "max_pages"), (dict(seqs=1 << 21), UNSUPPORTED, "sequences"),
    (dict(pts=-1), INVALID, "page_table_stride"),
])
def test_attention_refusals(args, code, text):
    from robustgemq_b200 import _lib

    a = dict(q=0x1000, qts=512, tokens=4, heads=4, table=0x1000, pts=8, pages=8, lens=0x1000, seqs=4, scale=1.0,
             window=0, out=0x1000) | args
    rc, msg = _status(_lib.load().gemq_paged_attention(
        ctypes.byref(_cache()), a["q"], a["qts"], a["tokens"], a["heads"], a["table"], a["pts"], a["pages"], a["lens"],
        None, a["seqs"], 0, 0, a["scale"], a["window"], a["out"], None, None, 0, None))
    assert rc == code and text in msg


def test_empty_calls_need_nothing():
    from robustgemq_b200 import _lib

    lib = _lib.load()
    ref = ctypes.byref(_cache())
    assert lib.gemq_kv_cache_write(ref, None, None, 0, 0, 0, 0, None, 0, None) == 0
    assert lib.gemq_kv_cache_read(ref, None, 0, None, None, None) == 0
    assert lib.gemq_paged_attention(ref, None, 0, 0, 4, None, 0, 0, None, None, 0, 0, 0, 1.0, 0, None, None, None, 0,
                                    None) == 0
    assert lib.gemq_verify_draft(ctypes.byref(_lib.VerifyT()), 0, 4, 100, None, 0, None) == 0


def _verify(**kw):
    from robustgemq_b200._lib import VerifyT

    v = VerifyT()
    v.logits = v.draft_tokens = v.uniforms = v.noise = v.tokens = v.num_accepted = v.logprobs = 0x1000
    for name, value in kw.items():
        setattr(v, name, value)
    return v


@pytest.mark.parametrize("change,sizes,ws,code,text", [
    ({}, (2, 0, 100), 1 << 20, INVALID, "num_drafts"), ({}, (2, 64, 100), 1 << 20, INVALID, "num_drafts"),
    ({}, (2, 3, 0), 1 << 20, INVALID, "vocab"), ({}, (70000, 3, 10), 1 << 20, UNSUPPORTED, "65535"),
    (dict(logits=None), (2, 3, 100), 1 << 20, INVALID, "null"), (dict(noise=None), (2, 3, 100), 1 << 20, INVALID, "null"),
    (dict(logits_dtype=5), (2, 3, 100), 1 << 20, INVALID, "dtype"),
    (dict(draft_probs=0x1000, probs_dtype=-1), (2, 3, 100), 1 << 20, INVALID, "dtype"),
    (dict(logits=0x1001), (2, 3, 100), 1 << 20, INVALID, "unaligned"),
    (dict(logits_row_stride=-1), (2, 3, 100), 1 << 20, INVALID, "stride"), ({}, (2, 3, 100), 8, WORKSPACE, "workspace"),
])
def test_verify_refusals(change, sizes, ws, code, text):
    from robustgemq_b200 import _lib

    rc, msg = _status(_lib.load().gemq_verify_draft(ctypes.byref(_verify(**change)), *sizes, 0x1000, ws, None))
    assert rc == code and text in msg


def test_python_entry_points_refuse_cpu_tensors_and_wrong_shapes():
    from robustgemq_b200 import serving

    k = torch.zeros((2, 1, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        serving.PagedKVCache.from_tensors(k, k)
    with pytest.raises(ValueError, match="bits"):
        serving.PagedKVCache(2, 16, 1, 64, bits=5, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        serving.verify_draft(torch.zeros((1, 2, 8)), torch.zeros((1, 1), dtype=torch.int64), torch.zeros((1, 1)),
                             torch.ones((1, 8)))


def test_plain_forms_agree_with_themselves():
    """The oracle's own checks: codes stay in range and within half a step, and a planted
    rejection changes the verified tokens."""
    x = np.random.default_rng(0).standard_normal((50, 64)).astype(np.float16)
    for bits, top in ((8, 127), (4, 15)):
        codes, step, base = quantise_rows(x, bits)
        assert codes.max() <= top and codes.min() >= (-127 if bits == 8 else 0)
        back = codes * step[:, None] + base[:, None]
        assert (np.abs(back - x) <= step[:, None] * 0.5001).all()
    logits = np.zeros((1, 3, 4))
    logits[0, :, 2] = 5.0
    drafts, noise = np.array([[2, 2]]), np.ones((1, 4))
    tokens, accepted, _, _ = verify_plain(logits, drafts, np.zeros((1, 2)), noise)
    assert tokens.tolist() == [[2, 2, 2]] and accepted.tolist() == [2]
    tokens, accepted, _, _ = verify_plain(logits, drafts, np.array([[0.0, 0.9999]]), noise)
    assert accepted.tolist() == [1] and tokens[0, 1] != 2 and tokens[0, 2] == -1


def test_lookup_draft_finds_the_latest_continuation():
    from robustgemq_b200.inference.speculative import lookup_draft

    assert lookup_draft([1, 2, 3, 9, 1, 2, 3, 4, 5, 1, 2, 3], 2) == [4, 5]
    assert lookup_draft([1, 2, 3, 9, 1, 2, 3], 10) == [9, 1, 2, 3]
    assert lookup_draft([5, 6, 7, 6], 3) == [7, 6]
    assert lookup_draft([1, 2, 3], 3) == [] and lookup_draft([1], 3) == [] and lookup_draft([], 3) == []
    assert lookup_draft([4, 4], 0) == []
