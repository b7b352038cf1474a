"""Plain 64-bit forms of the serving operators, and the inputs their tests share."""

from __future__ import annotations

import math

import numpy as np
import torch

# unit roundoff: half the distance between 1 and the next value
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def quantise_rows(x, bits):
    """Codes, step, base of rows ``x`` (numpy, any leading shape) by the stored forms'
    definition, in the float32 operations the definition names."""
    x = np.asarray(x, dtype=np.float32)
    tiny = np.float32(2.0 ** -64)
    if bits == 8:
        m = np.maximum(np.abs(x).max(-1), np.float32(127) * tiny)
        codes = np.rint(x * np.float32(127) / m[..., None])
        return codes, m / np.float32(127), np.zeros_like(m)
    lo = x.min(-1)
    r = np.maximum(x.max(-1) - lo, np.float32(15) * tiny)
    codes = np.rint((x - lo[..., None]) * np.float32(15) / r[..., None])
    return codes, r / np.float32(15), lo


def stored_values(x, bits):
    """What rows ``x`` read back as, before their rounding to 16 bits."""
    if bits == 16:
        return np.asarray(x, dtype=np.float64)
    codes, step, base = quantise_rows(x, bits)
    return codes.astype(np.float64) * step[..., None].astype(np.float64) + base[..., None].astype(np.float64)


def make_cache(pages, page, heads, dim, bits, dtype, layout="own", device="cuda"):
    """A cache whose every byte is poison: NaN rows (16 bits) or NaN steps. ``layout``:
    own tensors; "pool": K and V of two layers interleaved in one pool; "tokens_first":
    [pages, page, heads, dim] in memory."""
    from robustgemq_b200.serving import PagedKVCache

    width = dim // 2 if bits == 4 else dim
    kind = {16: dtype, 8: torch.int8, 4: torch.uint8}[bits]
    fill = float("nan") if bits == 16 else 85

    def rows():
        if layout == "pool":
            pool = torch.full((pages, 4, heads, page, width), fill, dtype=kind, device=device)
            return pool[:, 2], pool[:, 3]
        if layout == "tokens_first":
            return tuple(torch.full((pages, page, heads, width), fill, dtype=kind, device=device).transpose(1, 2)
                         for _ in range(2))
        return tuple(torch.full((pages, heads, page, width), fill, dtype=kind, device=device) for _ in range(2))

    k, v = rows()
    if bits == 16:
        return PagedKVCache.from_tensors(k, v)
    shape = (pages, heads, page) if bits == 8 else (pages, heads, page, 2)
    ks, vs = (torch.full(shape, float("nan"), device=device) for _ in range(2))
    return PagedKVCache.from_tensors(k, v, ks, vs, dtype=dtype)


class Batch:
    """Sequences with (new tokens, length) ``lens``, their cache written through
    ``PagedKVCache.write`` and the 64-bit values it then holds."""

    def __init__(self, lens, heads, kv_heads, dim, page, bits, dtype, seed=0, layout="own", spare=3, q_gain=1.5):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.dtype, self.bits, self.page = lens, dtype, bits, page
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        need = [-(-length // page) for _, length in lens]
        total = sum(need) + spare
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        width = max(max(need), 1)
        # entries past a sequence's last page are never read: a page id that does not exist
        self.page_table = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.page_table[b, :n] = order[at:at + n]
            at += n
        self.page_table = self.page_table.cuda()
        self.kv_lens = torch.tensor([length for _, length in lens], dtype=torch.int32, device="cuda")
        starts = np.concatenate([[0], np.cumsum([n for n, _ in lens])])
        self.q_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.tokens = int(starts[-1])
        self.cache = make_cache(total, page, kv_heads, dim, bits, dtype, layout)
        self.q = (torch.randn((self.tokens, heads, dim), generator=gen, device="cuda") * q_gain).to(dtype)
        self.k, self.v = [], []
        for b, (_, length) in enumerate(lens):
            k = torch.randn((length, kv_heads, dim), generator=gen, device="cuda").to(dtype)
            v = torch.randn((length, kv_heads, dim), generator=gen, device="cuda").to(dtype)
            self.put(b, torch.arange(length, device="cuda"), k, v)
            self.k.append(torch.from_numpy(stored_values(k.float().cpu().numpy(), bits)).cuda())
            self.v.append(torch.from_numpy(stored_values(v.float().cpu().numpy(), bits)).cuda())

    def slots(self, b, positions):
        return self.page_table[b, positions // self.page].long() * self.page + positions % self.page

    def put(self, b, positions, k, v):
        if len(positions):
            self.cache.write(k, v, self.slots(b, positions))

    def expect(self, scale, window=0):
        """(out, lse, bound on out, bound on lse), float64.

        Bound: the fp32 dot product of D terms is off by at most D 2^-23 sum |q k| (a
        tensor core may truncate, hence not 2^-24), which moves every weight by that
        (relatively, twice as it enters numerator and denominator); a weight rounded to 16
        bits moves by its roundoff u, or 2^-25 of the row's largest where fp16 runs out of
        exponent; sums of n weights in fp32 by n 2^-23 at most; the output is rounded
        once: u |o|."""
        outs, lses, tols, ltols = [], [], [], []
        at = 0
        u = ROUND[self.dtype]
        for b, (n, length) in enumerate(self.lens):
            q = self.q[at:at + n].double()
            at += n
            if n == 0:
                continue
            g = self.heads // self.kv_heads
            k = self.k[b].repeat_interleave(g, 1)
            v = self.v[b].repeat_interleave(g, 1)
            pos = torch.arange(length - n, length, device="cuda")[:, None]
            key = torch.arange(length, device="cuda")[None]
            seen = key <= pos
            if window:
                seen &= key > pos - window
            s = torch.einsum("qhd,khd->hqk", q, k) * scale
            mag = torch.einsum("qhd,khd->hqk", q.abs(), k.abs()) * abs(scale)
            s = torch.where(seen, s, torch.full_like(s, -math.inf))
            if length:
                m = s.amax(-1, keepdim=True)
                m = torch.where(m == -math.inf, torch.zeros_like(m), m)
                e = torch.where(seen, torch.exp(s - m), torch.zeros_like(s))
                z = e.sum(-1, keepdim=True)
                p = e / torch.where(z == 0, torch.ones_like(z), z)
                lse = (m + z.log())[..., 0]
                vs = torch.where(seen.any(0)[:, None, None], v, torch.zeros_like(v))
                o = torch.einsum("hqk,khd->qhd", p, vs)
                a = torch.einsum("hqk,khd->qhd", p, vs.abs())
                ds = torch.where(seen, mag, torch.zeros_like(mag)).amax(-1) * self.dim * 2.0 ** -23  # [h, q]
                top = p.amax(-1)  # [h, q]
            else:
                o = torch.zeros((n, self.heads, self.dim), dtype=torch.float64, device="cuda")
                a, vs = torch.zeros_like(o), torch.zeros((1, 1, 1), dtype=torch.float64, device="cuda")
                lse = torch.full((self.heads, n), -math.inf, dtype=torch.float64, device="cuda")
                ds = top = torch.zeros_like(lse)
            sums = length * 2.0 ** -23
            tiny = length * 2.0 ** -25 * top.T[..., None] * vs.abs().amax()
            outs.append(o)
            lses.append(lse.T)
            tols.append(u * (o.abs() + a) * 1.01 + (2 * ds.T[..., None] + sums + 2.0 ** -20) * a + tiny + 2.0 ** -24)
            ltols.append(ds.T + sums + 2.0 ** -20 * (1 + lse.T.abs().nan_to_num(posinf=0.0)))
        return torch.cat(outs), torch.cat(lses), torch.cat(tols), torch.cat(ltols)

    def check(self, scale=None, window=0, max_q_len=0, max_kv_len=0, use_starts=True):
        from robustgemq_b200.serving import paged_attention

        scale = self.dim ** -0.5 if scale is None else scale
        out, lse = paged_attention(self.q, self.cache, self.page_table, self.kv_lens,
                                   q_starts=self.q_starts if use_starts else None, max_q_len=max_q_len,
                                   max_kv_len=max_kv_len, scale=scale, window=window, return_lse=True)
        o, e, tol, ltol = self.expect(scale, window)
        assert out.dtype == self.dtype and out.shape == self.q.shape
        bad = ~((out.double() - o).abs() <= tol)
        assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outputs off, first at {bad.nonzero()[0].tolist()}, "
                               f"worst {float(((out.double() - o).abs() / tol).nan_to_num(1e9).max()):.3g} times the bound")
        empty = e == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        assert ((lse.double() - e).abs()[~empty] <= ltol[~empty]).all()
        return out, lse


def verify_plain(logits, drafts, uniforms, noise, probs=None, lens=None, temps=None):
    """(tokens, accepted, logprobs, margin) by the definition in float64; ``margin [B]``:
    the smallest relative distance of a decision to its other outcome."""
    B, rows, V = logits.shape
    n = rows - 1
    tokens = np.full((B, n + 1), -1, dtype=np.int64)
    accepted = np.zeros(B, dtype=np.int32)
    lp = np.zeros((B, n + 1))
    margin = np.full(B, np.inf)
    for b in range(B):
        t = 1.0 if temps is None else float(temps[b])
        count = n if lens is None else int(lens[b])
        for i in range(n + 1):
            row = logits[b, i].astype(np.float64)
            ok_row = not (np.isnan(row).any() or (row == np.inf).any() or not np.isfinite(row).any()) and t >= 0
            if ok_row:
                x = row / (t or 1.0)
                logs = x - x.max() - np.log(np.exp(x - x.max()).sum())
                p = np.exp(logs)
                if t == 0:
                    p = (np.arange(V) == row.argmax()).astype(np.float64)
            q = np.zeros(V)
            if i < count:
                d = int(drafts[b, i])
                if probs is not None:
                    q = probs[b, i].astype(np.float64)
                elif 0 <= d < V:
                    q[d] = 1.0
                if ok_row and 0 <= d < V:
                    left, right = float(uniforms[b, i]) * q[d], p[d]
                    if max(left, right) > 0 and 0 < t:
                        margin[b] = min(margin[b], abs(left - right) / max(left, right))
                    if left < right:
                        tokens[b, i], lp[b, i] = d, logs[d]
                        accepted[b] += 1
                        continue
            if ok_row:
                w = np.maximum(p - q, 0)
                # how far rounding may move a difference's score
                blur = 1e-5 * np.maximum(p, q) / noise[b].astype(np.float64) * (t > 0)
                if not (w > 0).any():
                    w = p
                score = np.where(w > 0, w / noise[b].astype(np.float64), -1)
                j = int(score.argmax())
                rest = np.delete(score, j)
                if len(rest) and rest.max() > 0 and t > 0:
                    margin[b] = min(margin[b], (score[j] - rest.max()) / score[j])
                if i < count and len(rest) and score[j] - blur[j] <= np.delete(score + blur, j).max():
                    margin[b] = 0.0  # a difference without digits left might win
                tokens[b, i], lp[b, i] = j, logs[j]
            break
    return tokens, accepted, lp, margin
