"""Several sequences decoded together from one paged cache, several tokens a step.

``PagedDecoder`` runs an OLMoE-shaped model (``generate.synthetic_olmoe`` or another
transformers model whose layers hold ``FusedOlmoeAttention``) on the serving operators
(``robustgemq_b200.serving``). Each step the sequences' new tokens, a prompt's chunk or the
last token and some drafted ones, go through the model as one batch of rows; every layer
writes their keys and values into its ``PagedKVCache`` (16, 8 or 4 bits) and attends over
the pages, and ``verify_draft`` decides which drafts stand. Drafts are looked up: what
followed the last tokens where they occurred before in the sequence itself. They cost no
model, and where nothing is found a step decodes one token as usual.

The reference's loop (gemq/benchmark_generate.py:113-156) decodes one sequence a token at a
time from a static fp16 cache and has no counterpart.
"""

from __future__ import annotations

import math
from typing import List, Optional, Sequence

import torch
from torch import Tensor

from .. import _lib
from ..serving import PagedKVCache, Verified, paged_attention, verify_draft
from .generate import FusedOlmoeAttention


def lookup_draft(tokens: Sequence[int], most: int, longest: int = 3) -> List[int]:
    """Up to ``most`` tokens that followed the latest earlier occurrence of the last
    ``longest`` tokens (or fewer, down to one) of ``tokens``."""
    n = len(tokens)
    for k in range(min(longest, n - 1), 0, -1):
        tail = list(tokens[n - k:])
        for i in range(n - k - 1, -1, -1):
            if list(tokens[i:i + k]) == tail:
                return list(tokens[i + k:i + k + most])
    return []


def _drawn(token: int) -> int:
    """The token that the verification drew, where it drew one."""
    if token < 0:
        raise RuntimeError("a row of logits has no distribution (a NaN, a +inf or nothing finite)")
    return token


class PagedDecoder:
    """Sequences of one model on paged caches, one a layer, that share a page table."""

    def __init__(self, model, num_pages: int, page_size: int = 64, bits: int = 8, max_pages_per_seq: int = 0):
        layers = model.model.layers
        for layer in layers:
            if not isinstance(layer.self_attn, FusedOlmoeAttention):
                raise ValueError("the model's layers must hold FusedOlmoeAttention (synthetic_olmoe(fused_attention=True))")
        att = layers[0].self_attn
        self.model = model
        self.device = next(model.parameters()).device
        self.head_dim = att.head_dim
        self.heads = model.config.num_attention_heads
        self.kv_heads = model.config.num_key_value_heads
        if self.kv_heads != self.heads:
            raise ValueError("the fused query, key and value projection has as many KV heads as heads")
        self.vocab = model.model.embed_tokens.weight.shape[0]
        self.page_size = page_size
        self.caches = [PagedKVCache(num_pages, page_size, self.kv_heads, self.head_dim, bits=bits,
                                    dtype=torch.float16, device=self.device) for _ in layers]
        self.free = list(range(num_pages - 1, -1, -1))
        self.width = max_pages_per_seq or num_pages
        self.pages: List[List[int]] = []   # of each sequence
        self.lengths: List[int] = []       # positions in the cache
        self.idle: List[int] = []          # released numbers, to be given out again
        self.page_table = torch.zeros((0, self.width), dtype=torch.int32, device=self.device)

    def add_sequence(self) -> int:
        """A new empty sequence; returns its number (a released one, where there is one)."""
        if self.idle:
            return self.idle.pop()
        self.pages.append([])
        self.lengths.append(0)
        row = torch.zeros((1, self.width), dtype=torch.int32, device=self.device)
        self.page_table = torch.cat([self.page_table, row])
        return len(self.pages) - 1

    def _reserve(self, seq: int, length: int) -> None:
        """Pages for the first ``length`` positions of a sequence."""
        need = -(-length // self.page_size) - len(self.pages[seq])
        if need <= 0:
            return
        if need > len(self.free) or len(self.pages[seq]) + need > self.width:
            raise RuntimeError("the paged cache is full")
        at = len(self.pages[seq])
        new = [self.free.pop() for _ in range(need)]
        self.pages[seq] += new
        self.page_table[seq, at:at + need] = torch.tensor(new, dtype=torch.int32, device=self.device)

    @torch.no_grad()
    def forward(self, seqs: Sequence[int], chunks: Sequence[Sequence[int]]) -> Tensor:
        """The model on ``chunks[i]``, the next tokens of sequence ``seqs[i]``, written to
        the cache at the positions after its length (which does not move: see
        ``advance``). Logits fp16 ``[sum of the chunks' lengths, vocab]``."""
        counts = [len(c) for c in chunks]
        if not counts or min(counts) < 1 or len(counts) != len(seqs):
            raise ValueError("one chunk of at least one token a sequence")
        if len(set(seqs)) != len(seqs) or not all(0 <= s < len(self.pages) for s in seqs):
            raise ValueError("sequences must be numbers of add_sequence, each once a call")
        if not all(0 <= t < self.vocab for c in chunks for t in c):
            raise ValueError(f"a token outside the vocabulary of {self.vocab}")
        self.idle = [s for s in self.idle if s not in seqs]  # (a released sequence, begun anew)
        lens = [self.lengths[s] + n for s, n in zip(seqs, counts)]
        for s, n in zip(seqs, lens):
            self._reserve(s, n)
        dev = self.device
        ids = torch.tensor([t for c in chunks for t in c], device=dev)
        pos = torch.cat([torch.arange(n - k, n) for n, k in zip(lens, counts)]).to(dev)
        row = torch.repeat_interleave(torch.tensor(list(seqs)), torch.tensor(counts)).to(dev)
        slots = self.page_table[row, pos // self.page_size].long() * self.page_size + pos % self.page_size
        starts = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=dev)
        kv_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        table = self.page_table[torch.tensor(list(seqs), device=dev)]
        m = self.model.model
        h = m.embed_tokens(ids)
        cos, sin = m.rotary_emb(h[None], pos[None])
        cos, sin = cos[0].half().contiguous(), sin[0].half().contiguous()
        for layer, cache in zip(m.layers, self.caches):
            x = self._attention(layer.self_attn, cache, layer.input_layernorm(h), cos, sin, slots, table, kv_lens, starts,
                                max(counts), max(lens))
            h = h + x
            h = h + layer.mlp(layer.post_attention_layernorm(h)[None])[0]
        return self.model.lm_head(m.norm(h))

    def _attention(self, att, cache, x, cos, sin, slots, table, kv_lens, starts, max_q_len, max_kv_len):
        qkv = att.qkv_proj(x)  # [rows, 3 n]
        rows, n = qkv.shape[0], qkv.shape[1] // 3
        q = torch.empty((rows, n), dtype=torch.float16, device=qkv.device)
        k = torch.empty_like(q)
        _lib.check(_lib.load().gemq_qk_norm_rope(
            _lib.ptr(qkv), qkv.stride(0), rows, n, self.head_dim, _lib.ptr(att.q_norm_weight), _lib.ptr(att.k_norm_weight),
            att.eps, _lib.ptr(cos), _lib.ptr(sin), _lib.ptr(q), _lib.ptr(k), None, None, 0, None,
            _lib.stream_ptr(qkv.device)))
        shape = (rows, self.heads, self.head_dim)
        cache.write(k.view(shape), qkv[:, 2 * n:].unflatten(1, shape[1:]), slots)
        out = paged_attention(q.view(shape), cache, table, kv_lens, q_starts=starts, max_q_len=max_q_len,
                              max_kv_len=max_kv_len, scale=float(att.scaling))
        return att.o_proj(out.view(rows, n))

    def advance(self, seq: int, tokens: int) -> None:
        """The first ``tokens`` of a sequence's last chunk stay in the cache; what came after
        them is overwritten by the next chunk."""
        self.lengths[seq] += tokens

    def release(self, seq: int) -> None:
        """Gives a sequence's pages back, and its number to the next new sequence."""
        self.free += reversed(self.pages[seq])
        self.pages[seq] = []
        self.lengths[seq] = 0
        if seq not in self.idle:
            self.idle.append(seq)

    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int, drafts: int = 4,
                 temperature: float = 0.0, chunk: int = 512, generator: Optional[torch.Generator] = None):
        """Continues every prompt by ``max_new_tokens`` tokens, greedily or sampled at
        ``temperature``, with up to ``drafts`` looked-up tokens a step. Returns the new
        tokens of each prompt and ``{"steps", "drafted", "accepted"}``. A row of logits without
        a distribution (a NaN, a +inf, nothing finite) is an error."""
        if not (0 <= temperature < math.inf):
            raise ValueError("temperature must be finite and not negative")
        if max_new_tokens < 0 or drafts < 0 or chunk < 1:
            raise ValueError("max_new_tokens and drafts must not be negative, chunk must be positive")
        if not all(len(p) for p in prompts):
            raise ValueError("a prompt needs at least one token")
        if len(prompts) == 0 or max_new_tokens == 0:
            return [[] for _ in prompts], {"steps": 0, "drafted": 0, "accepted": 0}
        seqs: List[int] = []
        try:
            for _ in prompts:
                seqs.append(self.add_sequence())
            return self._continue(seqs, prompts, max_new_tokens, drafts, float(temperature), chunk, generator)
        finally:
            for s in seqs:
                self.release(s)

    def _continue(self, seqs, prompts, max_new_tokens, drafts, temperature, chunk, generator):
        tokens = [list(p) for p in prompts]
        dev = self.device
        last: List[Optional[Tensor]] = [None] * len(seqs)
        for i, s in enumerate(seqs):  # prompts, in chunks
            for at in range(0, len(tokens[i]), chunk):
                part = tokens[i][at:at + chunk]
                last[i] = self.forward([s], [part])[-1]
                self.advance(s, len(part))
        vocab = last[0].shape[-1]

        def noise(n):
            return torch.empty((n, vocab), device=dev).exponential_(generator=generator)

        temps = torch.full((len(seqs),), temperature, device=dev)
        # the first token: one draft that counts for nothing, so that the race decides
        none = torch.zeros((len(seqs),), dtype=torch.int32, device=dev)
        first = verify_draft(torch.stack(last)[:, None].expand(-1, 2, -1).contiguous(), none[:, None].long(),
                             torch.zeros((len(seqs), 1), device=dev), noise(len(seqs)), draft_lens=none, temperature=temps)
        for i, t in enumerate(first.tokens[:, 0].tolist()):
            tokens[i].append(_drawn(t))
        stats = {"steps": 0, "drafted": 0, "accepted": 0}
        done = [len(p) + max_new_tokens for p in prompts]
        while True:
            live = [i for i in range(len(seqs)) if len(tokens[i]) < done[i]]
            if not live:
                break
            guess = [lookup_draft(tokens[i], min(drafts, done[i] - len(tokens[i]) - 1)) for i in live]
            width = max(1, max(len(g) for g in guess))
            logits = self.forward([seqs[i] for i in live], [[tokens[i][-1]] + g for i, g in zip(live, guess)])
            r = self._verify(logits, guess, width, temps[live], noise(len(live)), generator)
            taken = r.num_accepted.tolist()
            out = r.tokens.tolist()
            for i, g, a, row in zip(live, guess, taken, out):
                tokens[i] += row[:a] + [_drawn(row[a])]
                self.advance(seqs[i], a + 1)
                stats["drafted"] += len(g)
                stats["accepted"] += a
            stats["steps"] += 1
        return [t[len(p):] for t, p in zip(tokens, prompts)], stats

    def _verify(self, logits, guess, width, temps, noise, generator) -> Verified:
        """``verify_draft`` on the packed rows of chunks of 1 + len(guess) tokens."""
        dev = self.device
        n = len(guess)
        first, at = [], 0
        for g in guess:
            first.append(at)
            at += 1 + len(g)
        idx = torch.tensor([[f + min(j, len(g)) for j in range(width + 1)] for f, g in zip(first, guess)], device=dev)
        draft = torch.tensor([g + [0] * (width - len(g)) for g in guess], dtype=torch.int64, device=dev)
        lens = torch.tensor([len(g) for g in guess], dtype=torch.int32, device=dev)
        u = torch.rand((n, width), device=dev, generator=generator)
        return verify_draft(logits[idx], draft, u, noise, draft_lens=lens, temperature=temps)
