"""Serving operators: what several sequences that decode together need next to the MoE
blocks (the reference's loop, gemq/benchmark_generate.py:113-156, keeps one sequence's
fp16 cache and has no counterpart).

``PagedKVCache``      one layer's keys and values in pages that sequences share, at 16, 8
                      or 4 bits; rows are quantised as they are written and can be read back
``paged_attention``   attention of a chunk of new tokens (one token: a decode step; a few:
                      drafted tokens; many: a prompt's chunk) over the cache
``verify_draft``      which drafted tokens the target accepts, and the token after them

All run on the current stream of the tensors' device, allocate outputs and workspaces
with ``torch.empty`` and raise on arguments they do not take. What only the device can
see (a slot past the cache, a length past the page table, a page id outside the cache)
is skipped or clamped and recorded in the device error word (``_lib.device_error``).
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from ._lib import KvCacheT, VerifyT, check

_CODES = {torch.float16: _lib.FP16, torch.bfloat16: _lib.BF16, torch.float32: _lib.FP32}


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _on(device: torch.device):
    """Context in which ``device`` is current (nothing to do when it is)."""
    return torch.cuda.device(device)


class PagedKVCache:
    """Keys and values of one layer: ``num_pages`` pages of ``page_size`` tokens, each with
    ``num_kv_heads`` rows of ``head_dim`` values. Token ``i`` of page ``p`` is slot
    ``p * page_size + i``; which pages a sequence has is the caller's page table.

    ``bits`` 16 keeps the rows as they are; 8 keeps int8 codes with one float32 step a row
    (symmetric); 4 keeps two codes a byte with a float32 step and the value of code 0 a row.
    ``dtype`` (float16 or bfloat16) is the type of the rows written and read, of queries
    and of attention outputs.

    Tensors: ``k``, ``v`` ``[num_pages, num_kv_heads, page_size, head_dim]`` (bits 4:
    uint8 with ``head_dim / 2`` last), ``k_scale``, ``v_scale`` float32 ``[num_pages,
    num_kv_heads, page_size]`` (bits 4: ``[..., 2]``). ``from_tensors`` takes any strides
    between pages, heads and tokens, so the tensors may be views of one pool.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, bits: int = 16,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        _need(bits in (16, 8, 4), "bits must be 16, 8 or 4")
        _need(min(num_pages, page_size, num_kv_heads, head_dim) > 0, "sizes must be positive")
        shape = (num_pages, num_kv_heads, page_size, head_dim // 2 if bits == 4 else head_dim)
        kind = {16: dtype, 8: torch.int8, 4: torch.uint8}[bits]
        sshape = None if bits == 16 else shape[:3] if bits == 8 else shape[:3] + (2,)

        def rows():
            return torch.zeros(shape, dtype=kind, device=device)

        def scales():
            return None if sshape is None else torch.zeros(sshape, dtype=torch.float32, device=device)

        self._bind(rows(), rows(), scales(), scales(), dtype)

    @classmethod
    def from_tensors(cls, k: Tensor, v: Tensor, k_scale: Optional[Tensor] = None, v_scale: Optional[Tensor] = None,
                     dtype: Optional[torch.dtype] = None) -> "PagedKVCache":
        """A cache over tensors the caller owns. The codes' type gives the bits (int8: 8,
        uint8: 4, else 16); ``dtype`` may be left out for 16 bits."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale, dtype if dtype is not None else k.dtype)
        return self

    def _bind(self, k, v, k_scale, v_scale, dtype):
        _need(k.is_cuda, "k must be a CUDA tensor (no CPU path)")
        _need(k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and k.dtype == v.dtype,
              "k and v must be alike: [num_pages, num_kv_heads, page_size, head_dim]")
        bits = 8 if k.dtype == torch.int8 else 4 if k.dtype == torch.uint8 else 16
        _need(dtype in (torch.float16, torch.bfloat16), "dtype must be float16 or bfloat16")
        _need(bits != 16 or k.dtype == dtype, "a 16-bit cache holds its dtype")
        strides = k.stride()
        _need(strides[3] == 1, "rows must be contiguous")
        pages, heads, page, width = k.shape
        c = KvCacheT()
        c.k, c.v = k.data_ptr(), v.data_ptr()
        size = k.element_size()
        c.strides = (strides[0] * size, strides[1] * size, strides[2] * size)
        devices = [v.device]
        if bits == 16:
            _need(k_scale is None and v_scale is None, "a 16-bit cache has no scales")
        else:
            want = k.shape[:3] if bits == 8 else k.shape[:3] + (2,)
            _need(k_scale is not None and v_scale is not None and k_scale.dtype == v_scale.dtype == torch.float32
                  and k_scale.shape == v_scale.shape == want and k_scale.stride() == v_scale.stride(),
                  f"k_scale and v_scale must be float32 {tuple(want)} with the same strides")
            ss = k_scale.stride()
            _need(bits == 8 or ss[3] == 1, "a row's step and base must be neighbours")
            c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            c.scale_strides = ss[:3]
            devices += [k_scale.device, v_scale.device]
        _need(all(d == k.device for d in devices), "all tensors of a cache must be on one device")
        c.num_pages, c.kv_heads, c.page_size = pages, heads, page
        c.head_dim = width * 2 if bits == 4 else width
        c.bits, c.dtype = bits, _CODES[dtype]
        self.k, self.v, self.k_scale, self.v_scale, self.dtype = k, v, k_scale, v_scale, dtype
        self.bits, self.num_pages, self.num_kv_heads, self.page_size = bits, pages, heads, page
        self.head_dim, self.device = c.head_dim, k.device
        self._c = c
        self._ref = ctypes.byref(c)

    def _check_rows(self, t: Tensor, name: str, tokens: int) -> Tensor:
        _need(t.dtype == self.dtype and t.device == self.device, f"{name} must be {self.dtype} on the cache's device")
        _need(t.dim() == 3 and t.shape == (tokens, self.num_kv_heads, self.head_dim),
              f"{name} must be [tokens, num_kv_heads, head_dim]")
        st = t.stride()
        # rows of another layout (a transposed view) are copied once
        if st[2] != 1 or st[0] % 8 or st[1] % 8 or st[0] < 0 or t.data_ptr() % 16:
            return t.contiguous()
        return t

    def _check_slots(self, slots: Tensor) -> Tensor:
        _need(slots.dtype == torch.int64 and slots.dim() == 1 and slots.device == self.device,
              "slots must be int64 [tokens] on the cache's device")
        return slots.contiguous()

    def write(self, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """Quantises token ``t``'s rows ``k[t]``, ``v[t]`` (``[tokens, num_kv_heads,
        head_dim]``) into slot ``slots[t]`` (int64). A negative slot skips its token. A row
        with a NaN or an infinity reads back as NaN throughout (8 and 4 bits)."""
        slots = self._check_slots(slots)
        tokens = slots.shape[0]
        k, v = self._check_rows(k, "k", tokens), self._check_rows(v, "v", tokens)
        ks, vs = k.stride(), v.stride()
        with _on(self.device):
            check(_lib.load().gemq_kv_cache_write(self._ref, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1],
                                                  slots.data_ptr(), tokens, _lib.stream_ptr(self.device)))

    def read(self, slots: Tensor) -> Tuple[Tensor, Tensor]:
        """The stored keys and values of ``slots``, ``[tokens, num_kv_heads, head_dim]`` in
        the cache's ``dtype``; zeros for a negative slot."""
        slots = self._check_slots(slots)
        tokens = slots.shape[0]
        shape = (2, tokens, self.num_kv_heads, self.head_dim)
        out = torch.empty(shape, dtype=self.dtype, device=self.device)
        k, v = out[0], out[1]
        with _on(self.device):
            check(_lib.load().gemq_kv_cache_read(self._ref, slots.data_ptr(), tokens, k.data_ptr(), v.data_ptr(),
                                                 _lib.stream_ptr(self.device)))
        return k, v


def paged_attention(q: Tensor, cache: PagedKVCache, page_table: Tensor, kv_lens: Tensor,
                    q_starts: Optional[Tensor] = None, max_q_len: int = 0, max_kv_len: int = 0,
                    scale: Optional[float] = None, window: int = 0,
                    return_lse: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Causal attention of new tokens over a cache that already holds their keys and values.

    ``q [tokens, q_heads, head_dim]``: the new tokens of all sequences one after another,
    sequence ``b``'s at ``q_starts[b]:q_starts[b + 1]`` (int32 ``[seqs + 1]``; left out:
    equally many each). ``kv_lens`` int32 ``[seqs]``: positions of each sequence, the new
    ones included. ``page_table`` int32 ``[seqs, pages]``: position ``j`` lies in page
    ``page_table[b, j // page_size]``. Query heads share KV heads in equal groups. Token
    ``i`` of ``n`` sees the positions up to ``kv_len - n + i``, with ``window > 0`` the last
    ``window`` of them; one that sees nothing gets zeros. Tokens outside every sequence are
    not written.

    ``max_q_len`` / ``max_kv_len``: the longest values the call may meet, if known (they
    choose kernel and split; 0 stands for all tokens and the whole table). ``scale``
    defaults to ``head_dim ** -0.5``. Returns ``out`` like ``q`` (contiguous), with
    ``return_lse`` also the natural log-sum-exp of the scaled scores, float32
    ``[tokens, q_heads]``.
    """
    dev = cache.device
    _need(q.dim() == 3 and q.dtype == cache.dtype and q.device == dev and q.shape[2] == cache.head_dim,
          "q must be [tokens, q_heads, head_dim] of the cache's dtype and device")
    _need(page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.device == dev,
          "page_table must be int32 [seqs, pages] on the cache's device")
    seqs, pages = page_table.shape
    _need(kv_lens.dtype == torch.int32 and kv_lens.shape == (seqs,) and kv_lens.device == dev,
          "kv_lens must be int32 [seqs] on the cache's device")
    if q_starts is not None:
        _need(q_starts.dtype == torch.int32 and q_starts.shape == (seqs + 1,) and q_starts.device == dev,
              "q_starts must be int32 [seqs + 1] on the cache's device")
        q_starts = q_starts.contiguous()
    kv_lens = kv_lens.contiguous()
    if page_table.stride(1) != 1 or page_table.stride(0) < 0:
        page_table = page_table.contiguous()
    tokens, heads, dim = q.shape
    st = q.stride()
    if st[2] != 1 or (st[1] != dim and heads != 1) or st[0] % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        st = q.stride()
    lib = _lib.load()
    out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=dev)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=dev) if return_lse else None
    with _on(dev):
        need = lib.gemq_paged_attention_workspace_size(cache._ref, tokens, heads, seqs, pages, max_q_len, max_kv_len)
        ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
        check(lib.gemq_paged_attention(
            cache._ref, q.data_ptr(), st[0], tokens, heads, page_table.data_ptr(), page_table.stride(0), pages,
            kv_lens.data_ptr(), None if q_starts is None else q_starts.data_ptr(), seqs, max_q_len, max_kv_len,
            dim ** -0.5 if scale is None else scale, window, out.data_ptr(), None if lse is None else lse.data_ptr(),
            None if ws is None else ws.data_ptr(), need, _lib.stream_ptr(dev)))
    return (out, lse) if return_lse else out


class Verified(NamedTuple):
    """``tokens`` int64 ``[seqs, drafts + 1]``: the accepted drafts, the token after them,
    then -1. ``num_accepted`` int32 ``[seqs]``. ``logprobs`` float32 ``[seqs, drafts + 1]``:
    the target's log probability of each token, 0 beside a -1."""

    tokens: Tensor
    num_accepted: Tensor
    logprobs: Tensor


def verify_draft(target_logits: Tensor, draft_tokens: Tensor, uniforms: Tensor, noise: Tensor,
                 draft_probs: Optional[Tensor] = None, draft_lens: Optional[Tensor] = None,
                 temperature: Optional[Tensor] = None) -> Verified:
    """Accepts or replaces drafted tokens so that what comes out is distributed as if the
    target had sampled it.

    ``target_logits [seqs, drafts + 1, vocab]`` (float16, bfloat16 or float32): the
    target's logits at the last known token and at every draft. ``draft_tokens`` int64
    ``[seqs, drafts]``, ``draft_lens`` int32 ``[seqs]`` how many of them count (all).
    ``draft_probs [seqs, drafts, vocab]``: what the draft sampled from; left out for drafts
    made without sampling. ``temperature`` float32 ``[seqs]`` (1; 0: greedy). The random
    numbers are given: ``uniforms`` float32 ``[seqs, drafts]`` in [0, 1) and ``noise``
    float32 ``[seqs, vocab]``, exponential (``torch.empty(...).exponential_()``).

    Draft ``x`` at position ``i`` is taken while ``uniforms * q(x) < p(x)``; then one token
    is drawn from ``max(p - q, 0)``, or from ``p`` after the last draft, as the largest of
    ``weight / noise`` (lowest index on ties). A row of logits with a NaN, a +inf or
    nothing finite takes no draft and gives the token -1.
    """
    _need(target_logits.is_cuda and target_logits.dim() == 3 and target_logits.dtype in _CODES,
          "target_logits must be a CUDA tensor [seqs, drafts + 1, vocab] of float16, bfloat16 or float32")
    dev = target_logits.device
    B, rows, V = target_logits.shape
    n = rows - 1
    _need(draft_tokens.dtype == torch.int64 and draft_tokens.shape == (B, n) and draft_tokens.device == dev,
          "draft_tokens must be int64 [seqs, drafts] beside target_logits")
    _need(uniforms.dtype == torch.float32 and uniforms.shape == (B, n) and uniforms.device == dev,
          "uniforms must be float32 [seqs, drafts] beside target_logits")
    _need(noise.dtype == torch.float32 and noise.shape == (B, V) and noise.device == dev,
          "noise must be float32 [seqs, vocab] beside target_logits")
    v = VerifyT()
    keep = []  # tensors whose copies the call reads

    def dense(t):
        t = t.contiguous()
        keep.append(t)
        return t.data_ptr()

    def strided(t):
        st = t.stride()
        if (st[2] != 1 and t.shape[2] != 1) or min(st) < 0:
            t = t.contiguous()
            keep.append(t)
            st = t.stride()
        return t.data_ptr(), st[0], st[1], _CODES[t.dtype]

    v.logits, v.logits_seq_stride, v.logits_row_stride, v.logits_dtype = strided(target_logits)
    if draft_probs is not None:
        _need(draft_probs.dtype in _CODES and draft_probs.shape == (B, n, V) and draft_probs.device == dev,
              "draft_probs must be [seqs, drafts, vocab] of float16, bfloat16 or float32 beside target_logits")
        v.draft_probs, v.probs_seq_stride, v.probs_row_stride, v.probs_dtype = strided(draft_probs)
    if draft_lens is not None:
        _need(draft_lens.dtype == torch.int32 and draft_lens.shape == (B,) and draft_lens.device == dev,
              "draft_lens must be int32 [seqs] beside target_logits")
        v.draft_lens = dense(draft_lens)
    if temperature is not None:
        _need(temperature.dtype == torch.float32 and temperature.shape == (B,) and temperature.device == dev,
              "temperature must be float32 [seqs] beside target_logits")
        v.temperature = dense(temperature)
    v.draft_tokens, v.uniforms, v.noise = dense(draft_tokens), dense(uniforms), dense(noise)
    tokens = torch.empty((B, n + 1), dtype=torch.int64, device=dev)
    accepted = torch.empty((B,), dtype=torch.int32, device=dev)
    logprobs = torch.empty((B, n + 1), dtype=torch.float32, device=dev)
    v.tokens, v.num_accepted, v.logprobs = tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr()
    lib = _lib.load()
    with _on(dev):
        need = lib.gemq_verify_draft_workspace_size(B, n, V)
        ws = torch.empty((need,), dtype=torch.uint8, device=dev)
        check(lib.gemq_verify_draft(ctypes.byref(v), B, n, V, ws.data_ptr(), need, _lib.stream_ptr(dev)))
    return Verified(tokens, accepted, logprobs)
