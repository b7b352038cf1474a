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

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from . import _lib
from . import build as _build

_lib.load()
_build.build_binding()  # where its sources are newer
from . import _serving_ext as _ext  # noqa: E402


class PagedKVCache(_ext.Cache):
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
        if bits not in (16, 8, 4):
            raise ValueError("bits must be 16, 8 or 4")
        if min(num_pages, page_size, num_kv_heads, head_dim) <= 0:
            raise ValueError("sizes must be positive")
        shape = (num_pages, num_kv_heads, page_size, head_dim // 2 if bits == 4 else head_dim)
        kind = {16: dtype, 8: torch.int8, 4: torch.uint8}[bits]
        sshape = None if bits == 16 else shape[:3] if bits == 8 else shape[:3] + (2,)

        def rows():
            return torch.zeros(shape, dtype=kind, device=device)

        def scales():
            return None if sshape is None else torch.zeros(sshape, dtype=torch.float32, device=device)

        super().__init__(rows(), rows(), scales(), scales(), dtype)

    @classmethod
    def from_tensors(cls, k: Tensor, v: Tensor, k_scale: Optional[Tensor] = None, v_scale: Optional[Tensor] = None,
                     dtype: Optional[torch.dtype] = None) -> "PagedKVCache":
        """A cache over tensors the caller owns. The codes' type gives the bits (int8: 8,
        uint8: 4, else 16); ``dtype`` may be left out for 16 bits."""
        self = cls.__new__(cls)
        _ext.Cache.__init__(self, k, v, k_scale, v_scale, k.dtype if dtype is None else dtype)
        return self

    def write(self, k: Tensor, v: Tensor, slots: Tensor) -> None:
        """Quantises token ``t``'s rows ``k[t]``, ``v[t]`` (``[tokens, num_kv_heads,
        head_dim]``) into slot ``slots[t]`` (int64). A negative slot skips its token; a slot
        given twice is left with parts of both tokens. At 8 and 4 bits a row reads back as
        NaN throughout where it has a NaN or an infinity, or where (bfloat16) 127 times its
        largest magnitude, or 15 times its range, leaves float32."""
        super().write(k, v, slots)

    def read(self, slots: Tensor) -> Tuple[Tensor, Tensor]:
        """The stored keys and values of ``slots``, ``[tokens, num_kv_heads, head_dim]`` in
        the cache's ``dtype``; zeros for a negative slot."""
        return super().read(slots)


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
    not written. At 8 and 4 bits a value row whose step is above 2^38 (bfloat16 values
    above 10^12) counts as NaN in the tokens that see it.

    ``max_q_len`` / ``max_kv_len``: the longest values the call may meet, if known. They
    choose kernel and split, and wrong ones cost time only; 0 stands for all tokens (without
    ``q_starts``: for as many as each sequence has) and the whole table. A batch of single
    or drafted tokens with ``q_starts`` and without ``max_q_len`` is taken for a prompt's
    chunk, several times slower than need be. ``scale``
    defaults to ``head_dim ** -0.5``. Returns ``out`` like ``q`` (contiguous), with
    ``return_lse`` also the natural log-sum-exp of the scaled scores, float32
    ``[tokens, q_heads]``.
    """
    out, lse = _ext.attention(q, cache, page_table, kv_lens, q_starts, max_q_len, max_kv_len, scale, window, return_lse)
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
    ``[seqs, drafts]``, ``draft_lens`` int32 ``[seqs]`` how many of them count (all; clamped
    to what there are).
    ``draft_probs [seqs, drafts, vocab]``: what the draft sampled from; left out for drafts
    made without sampling. ``temperature`` float32 ``[seqs]`` (1; 0: greedy). The random
    numbers are given: ``uniforms`` float32 ``[seqs, drafts]`` in [0, 1) and ``noise``
    float32 ``[seqs, vocab]``, exponential (``torch.empty(...).exponential_()``).

    Draft ``x`` at position ``i`` is taken while ``uniforms * q(x) < p(x)``; then one token
    is drawn from ``max(p - q, 0)``, or from ``p`` after the last draft, as the largest of
    ``weight / noise`` (lowest index on ties). A row of logits with a NaN, a +inf or
    nothing finite takes no draft and gives the token -1.
    """
    return Verified(*_ext.verify(target_logits, draft_tokens, uniforms, noise, draft_probs, draft_lens, temperature))
