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


# These calls are short: on small inputs the host's part of a call is its time. So the
# argument checks build no message unless they fail, and the stream and the current
# device are asked of torch directly.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else lambda: -1
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _run(index: int, fn, *args) -> None:
    """``fn(*args, stream)`` with device ``index`` current, on its current stream."""
    if _current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status)


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
        shape, strides, kind, dev = k.shape, k.stride(), k.dtype, k.device
        if not k.is_cuda:
            raise ValueError("k must be a CUDA tensor (no CPU path)")
        if len(shape) != 4 or v.shape != shape or v.stride() != strides or v.dtype != kind or v.device != dev:
            raise ValueError("k and v must be alike: [num_pages, num_kv_heads, page_size, head_dim] on one device")
        code = _CODES.get(dtype)
        if code is None or code == _lib.FP32:
            raise ValueError("dtype must be float16 or bfloat16")
        if strides[3] != 1:
            raise ValueError("rows must be contiguous")
        c = KvCacheT()
        pages, heads, page, dim = shape
        if kind is torch.int8 or kind is torch.uint8:
            bits, size = (8, 1) if kind is torch.int8 else (4, 1)
            want = shape[:3] if bits == 8 else shape[:3] + (2,)
            if k_scale is None or v_scale is None:
                raise ValueError("a quantised cache needs k_scale and v_scale")
            ss = k_scale.stride()
            if not (k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32 and k_scale.shape == want and
                    v_scale.shape == want and v_scale.stride() == ss and k_scale.device == dev and
                    v_scale.device == dev):
                raise ValueError(f"k_scale and v_scale must be float32 {tuple(want)} with the same strides, beside k")
            if bits == 4:
                if ss[3] != 1:
                    raise ValueError("a row's step and base must be neighbours")
                dim *= 2
            c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            c.scale_strides = ss[:3]
        else:
            bits, size = 16, 2
            if kind is not dtype:
                raise ValueError("a 16-bit cache holds its dtype")
            if k_scale is not None or v_scale is not None:
                raise ValueError("a 16-bit cache has no scales")
        c.k, c.v = k.data_ptr(), v.data_ptr()
        c.strides = (strides[0] * size, strides[1] * size, strides[2] * size)
        c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.bits, c.dtype = pages, heads, page, dim, bits, code
        self.k, self.v, self.k_scale, self.v_scale, self.dtype = k, v, k_scale, v_scale, dtype
        self.bits, self.num_pages, self.num_kv_heads, self.page_size = bits, pages, heads, page
        self.head_dim, self.device = dim, dev
        self._index = dev.index
        self._c = c
        self._ref = ctypes.byref(c)

    def _check_rows(self, t: Tensor, name: str, tokens: int) -> Tensor:
        if t.dtype is not self.dtype or t.device != self.device:
            raise ValueError(f"{name} must be {self.dtype} on the cache's device")
        if t.shape != (tokens, self.num_kv_heads, self.head_dim):
            raise ValueError(f"{name} must be [tokens, num_kv_heads, head_dim]")
        st = t.stride()
        # rows of another layout (a transposed view) are copied once
        if st[2] != 1 or st[0] % 8 or st[1] % 8 or t.data_ptr() % 16:
            return t.contiguous()
        return t

    def _check_slots(self, slots: Tensor) -> Tensor:
        if slots.dtype is not torch.int64 or slots.dim() != 1 or slots.device != self.device:
            raise ValueError("slots must be int64 [tokens] on the cache's device")
        return slots if slots.is_contiguous() else slots.contiguous()

    def write(self, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """Quantises token ``t``'s rows ``k[t]``, ``v[t]`` (``[tokens, num_kv_heads,
        head_dim]``) into slot ``slots[t]`` (int64). A negative slot skips its token. A row
        with a NaN or an infinity reads back as NaN throughout (8 and 4 bits)."""
        slots = self._check_slots(slots)
        tokens = slots.shape[0]
        k, v = self._check_rows(k, "k", tokens), self._check_rows(v, "v", tokens)
        ks, vs = k.stride(), v.stride()
        _run(self._index, _lib.load().gemq_kv_cache_write, self._ref, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0],
             vs[1], slots.data_ptr(), tokens)

    def read(self, slots: Tensor) -> Tuple[Tensor, Tensor]:
        """The stored keys and values of ``slots``, ``[tokens, num_kv_heads, head_dim]`` in
        the cache's ``dtype``; zeros for a negative slot."""
        slots = self._check_slots(slots)
        shape = (slots.shape[0], self.num_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=self.dtype, device=self.device)
        v = torch.empty(shape, dtype=self.dtype, device=self.device)
        _run(self._index, _lib.load().gemq_kv_cache_read, self._ref, slots.data_ptr(), shape[0], k.data_ptr(),
             v.data_ptr())
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
    tokens, heads, dim = shape = q.shape if q.dim() == 3 else (0, 0, -1)
    if q.dtype is not cache.dtype or q.device != dev or dim != cache.head_dim:
        raise ValueError("q must be [tokens, q_heads, head_dim] of the cache's dtype and device")
    if page_table.dim() != 2 or page_table.dtype is not torch.int32 or page_table.device != dev:
        raise ValueError("page_table must be int32 [seqs, pages] on the cache's device")
    seqs, pages = page_table.shape
    if kv_lens.dtype is not torch.int32 or kv_lens.shape != (seqs,) or kv_lens.device != dev:
        raise ValueError("kv_lens must be int32 [seqs] on the cache's device")
    starts = None
    if q_starts is not None:
        if q_starts.dtype is not torch.int32 or q_starts.shape != (seqs + 1,) or q_starts.device != dev:
            raise ValueError("q_starts must be int32 [seqs + 1] on the cache's device")
        q_starts = q_starts.contiguous()
        starts = q_starts.data_ptr()
    kv_lens = kv_lens.contiguous()
    ts = page_table.stride()
    if ts[1] != 1:
        page_table = page_table.contiguous()
        ts = page_table.stride()
    st = q.stride()
    if st[2] != 1 or (st[1] != dim and heads != 1) or st[0] % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        st = q.stride()
    lib = _lib.load()
    out = torch.empty(shape, dtype=q.dtype, device=dev)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=dev) if return_lse else None
    if cache._index != _current_device():
        with torch.cuda.device(cache._index):
            need = lib.gemq_paged_attention_workspace_size(cache._ref, tokens, heads, seqs, pages, max_q_len, max_kv_len)
    else:
        need = lib.gemq_paged_attention_workspace_size(cache._ref, tokens, heads, seqs, pages, max_q_len, max_kv_len)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _run(cache._index, lib.gemq_paged_attention, cache._ref, q.data_ptr(), st[0], tokens, heads, page_table.data_ptr(),
         ts[0], pages, kv_lens.data_ptr(), starts, seqs, max_q_len, max_kv_len, dim ** -0.5 if scale is None else scale,
         window, out.data_ptr(), None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), need)
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
    if not target_logits.is_cuda or target_logits.dim() != 3 or target_logits.dtype not in _CODES:
        raise ValueError("target_logits must be a CUDA tensor [seqs, drafts + 1, vocab] of float16, bfloat16 or float32")
    dev = target_logits.device
    B, rows, V = target_logits.shape
    n = rows - 1
    if draft_tokens.dtype is not torch.int64 or draft_tokens.shape != (B, n) or draft_tokens.device != dev:
        raise ValueError("draft_tokens must be int64 [seqs, drafts] beside target_logits")
    if uniforms.dtype is not torch.float32 or uniforms.shape != (B, n) or uniforms.device != dev:
        raise ValueError("uniforms must be float32 [seqs, drafts] beside target_logits")
    if noise.dtype is not torch.float32 or noise.shape != (B, V) or noise.device != dev:
        raise ValueError("noise must be float32 [seqs, vocab] beside target_logits")
    # (names bound to copies live until the call has been issued)
    v = VerifyT()
    st = target_logits.stride()
    if st[2] != 1:
        target_logits = target_logits.contiguous()
        st = target_logits.stride()
    v.logits, v.logits_seq_stride, v.logits_row_stride = target_logits.data_ptr(), st[0], st[1]
    v.logits_dtype = _CODES[target_logits.dtype]
    if draft_probs is not None:
        if draft_probs.dtype not in _CODES or draft_probs.shape != (B, n, V) or draft_probs.device != dev:
            raise ValueError("draft_probs must be [seqs, drafts, vocab] of float16, bfloat16 or float32 beside "
                             "target_logits")
        st = draft_probs.stride()
        if st[2] != 1:
            draft_probs = draft_probs.contiguous()
            st = draft_probs.stride()
        v.draft_probs, v.probs_seq_stride, v.probs_row_stride = draft_probs.data_ptr(), st[0], st[1]
        v.probs_dtype = _CODES[draft_probs.dtype]
    if draft_lens is not None:
        if draft_lens.dtype is not torch.int32 or draft_lens.shape != (B,) or draft_lens.device != dev:
            raise ValueError("draft_lens must be int32 [seqs] beside target_logits")
        draft_lens = draft_lens.contiguous()
        v.draft_lens = draft_lens.data_ptr()
    if temperature is not None:
        if temperature.dtype is not torch.float32 or temperature.shape != (B,) or temperature.device != dev:
            raise ValueError("temperature must be float32 [seqs] beside target_logits")
        temperature = temperature.contiguous()
        v.temperature = temperature.data_ptr()
    draft_tokens, uniforms, noise = draft_tokens.contiguous(), uniforms.contiguous(), noise.contiguous()
    v.draft_tokens, v.uniforms, v.noise = draft_tokens.data_ptr(), uniforms.data_ptr(), noise.data_ptr()
    tokens = torch.empty((B, rows), dtype=torch.int64, device=dev)
    accepted = torch.empty((B,), dtype=torch.int32, device=dev)
    logprobs = torch.empty((B, rows), dtype=torch.float32, device=dev)
    v.tokens, v.num_accepted, v.logprobs = tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr()
    lib = _lib.load()
    index = dev.index
    need = lib.gemq_verify_draft_workspace_size(B, n, V)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _run(index, lib.gemq_verify_draft, ctypes.byref(v), B, n, V, ws.data_ptr(), need)
    return Verified(tokens, accepted, logprobs)
