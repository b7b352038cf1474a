"""The serving operators' cases: a paged KV cache quantised as it is written and read
back, attention of a chunk of new tokens over it, and the verification of drafted
tokens. ``run`` makes a user's calls where ``own`` is true; else it computes the same
in plain torch operations in 32 bits. ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

FP16, BF16, FP32 = "fp16", "bf16", "fp32"
DTYPES = {FP16: torch.float16, BF16: torch.bfloat16, FP32: torch.float32}
ELEM = {FP16: 2, BF16: 2, FP32: 4}
MIN_SCALE = 2.0 ** -64  # the smallest scale a quantised row is stored with


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one new token of each of 64 running sequences, 16 KV heads: latency
        dict(name="append_8bit_b64", op="cache", tokens=64, heads=16, dim=128, page=16, bits=8, dtype=FP16),
        # a long prompt's keys and values at 4 bits, four KV heads
        dict(name="prompt_4bit_8k", op="cache", tokens=8192, heads=4, dim=128, page=64, bits=4, dtype=BF16),
        # many prompts at once, a head size that is no power of two, an odd token count
        dict(name="prompt_8bit_50k", op="cache", tokens=50001, heads=8, dim=80, page=32, bits=8, dtype=FP16),
        # one token of one sequence, 16 heads of their own keys: the smallest step
        dict(name="decode_b1", op="attention", seqs=1, q_len=1, kv_len=2048, ragged=0, heads=16, kv_heads=16, dim=128,
             page=16, bits=16, dtype=FP16, window=0, lse=False),
        # a full batch of running sequences of uneven lengths, eight query heads a KV head
        dict(name="decode_b64_8bit", op="attention", seqs=64, q_len=1, kv_len=8192, ragged=7, heads=32, kv_heads=4,
             dim=128, page=64, bits=8, dtype=FP16, window=0, lse=False),
        # four drafted tokens and the last one of 16 sequences, to be verified
        dict(name="draft_b16_4bit", op="attention", seqs=16, q_len=5, kv_len=4096, ragged=3, heads=16, kv_heads=16,
             dim=128, page=32, bits=4, dtype=FP16, window=0, lse=False),
        # two long documents, one token each: few rows, a long axis
        dict(name="decode_long_b2", op="attention", seqs=2, q_len=1, kv_len=131072, ragged=0, heads=32, kv_heads=8,
             dim=128, page=64, bits=16, dtype=BF16, window=0, lse=False),
        # the last chunk of a long prompt: the largest
        dict(name="chunk_4k_of_16k", op="attention", seqs=1, q_len=4096, kv_len=16384, ragged=0, heads=32, kv_heads=8,
             dim=128, page=128, bits=16, dtype=BF16, window=0, lse=False),
        # chunks of uneven lengths together, sliding window, 8 bits, smaller heads, with the log-sum-exp
        dict(name="chunks_mixed_8bit", op="attention", seqs=12, q_len=1000, kv_len=9000, ragged=11, heads=24,
             kv_heads=8, dim=64, page=32, bits=8, dtype=FP16, window=4096, lse=True),
        # four tokens proposed by lookup (no draft probabilities) for one sequence
        dict(name="verify_b1", op="verify", seqs=1, drafts=4, vocab=50304, dtype=FP16, probs="", ragged=0, temps="one"),
        # a full batch with a draft model's probabilities, a large vocabulary
        dict(name="verify_b64", op="verify", seqs=64, drafts=7, vocab=151936, dtype=BF16, probs=FP32, ragged=0,
             temps="one"),
        # uneven draft lengths, greedy and sampled sequences together, an odd vocabulary
        dict(name="verify_mixed", op="verify", seqs=24, drafts=5, vocab=32001, dtype=FP32, probs=FP16, ragged=5,
             temps="mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["cache", "attention", "attention", "verify"])
    if op == "cache":
        heads, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 80, 96, 128, 256])
        most = 50001 * 8 * 80 // (heads * dim)
        return dict(op=op, tokens=min(_log_int(rng, 1, 50000), most), heads=heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128]), bits=rng.choice([16, 8, 4]), dtype=rng.choice([FP16, BF16]))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
        dim = rng.choice([64, 80, 128, 128, 256])
        q_len = rng.choice([1, 1, rng.randint(2, 9), _log_int(rng, 10, 4096)])
        seqs = _log_int(rng, 1, 64)
        kv_len = max(q_len, _log_int(rng, 16, 131072))
        # no more score elements and cache than the largest listed cases have
        while seqs > 1 and (seqs * heads * q_len * kv_len > 1.5e9 or seqs * kv_heads * kv_len * dim > 2.6e8):
            seqs = (seqs + 1) // 2
        while heads * q_len * kv_len * dim > 32 * 4096 * 14336 * 128 or kv_heads * kv_len * dim > 2.6e8:
            kv_len = max(16, kv_len * 2 // 3)
            q_len = min(q_len, kv_len)
        return dict(op=op, seqs=seqs, q_len=q_len, kv_len=kv_len, ragged=rng.randint(1, 999), heads=heads,
                    kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]), bits=rng.choice([16, 8, 4]),
                    dtype=rng.choice([FP16, BF16]), window=rng.choice([0, 0, 0, rng.randint(1, 6000)]),
                    lse=rng.choice([False, True]))
    vocab = _log_int(rng, 1000, 151936)
    drafts = rng.randint(1, 8)
    return dict(op=op, seqs=min(_log_int(rng, 1, 64), 64 * 8 * 151936 // ((drafts + 1) * vocab)), drafts=drafts,
                vocab=vocab, dtype=rng.choice([FP16, BF16, FP32]), probs=rng.choice(["", FP16, FP32]),
                ragged=rng.choice([0, rng.randint(1, 999)]), temps=rng.choice(["one", "mixed"]))


def _lengths(case):
    """(new tokens, length with them) of each sequence: uneven where the case is ragged,
    the first one at the full size."""
    r = random.Random(case["ragged"])
    out = []
    for b in range(case["seqs"]):
        if not case["ragged"] or b == 0:
            out.append((case["q_len"], case["kv_len"]))
        else:
            n = r.randint(1, case["q_len"])
            out.append((n, max(n, r.randint(max(1, case["kv_len"] // 8), case["kv_len"]))))
    return out


def _draft_lengths(case):
    r = random.Random(case["ragged"])
    return [r.randint(0, case["drafts"]) if case["ragged"] else case["drafts"] for _ in range(case["seqs"])]


def _row_bytes(bits, dim):
    """Stored bytes of one token's key (or value) of one head, scales included."""
    return dim * bits // 8 + {16: 0, 8: 4, 4: 8}[bits]


def work(case):
    if case["op"] == "cache":
        rows = 2 * case["tokens"] * case["heads"]
        # read the input, write the cache, read the cache, write what was read; 8-byte slots twice
        return {"bytes": rows * (4 * case["dim"] + 2 * _row_bytes(case["bits"], case["dim"])) + 16 * case["tokens"],
                "flops": rows * 4 * case["dim"]}
    if case["op"] == "attention":
        nbytes = flops = 0
        for n, length in _lengths(case):
            w = case["window"] or length
            # query i sees min(length - n + i + 1, w) keys
            first, last = length - n + 1, length
            full = max(0, last - max(first, w) + 1)  # queries that see w keys
            part = n - full
            pairs = full * w + part * first + part * (part - 1) // 2
            seen = min(length, w + n - 1)
            nbytes += 2 * seen * case["kv_heads"] * _row_bytes(case["bits"], case["dim"])
            nbytes += n * case["heads"] * (4 * case["dim"] + (4 if case["lse"] else 0))
            flops += 4 * case["dim"] * case["heads"] * pairs
        return {"bytes": nbytes, "flops": flops}
    rows = sum(n + 1 for n in _draft_lengths(case))
    nbytes = rows * case["vocab"] * ELEM[case["dtype"]] + 4 * case["seqs"] * case["vocab"]
    if case["probs"]:
        nbytes += sum(1 for n in _draft_lengths(case) if n) * case["vocab"] * ELEM[case["probs"]]
    return {"bytes": nbytes, "flops": 4 * rows * case["vocab"]}


# ------------------------------------------------------------------ what the program has before the call
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    st = {"case": case}
    if case["op"] == "cache":
        T, H, D, page = case["tokens"], case["heads"], case["dim"], case["page"]
        dt = DTYPES[case["dtype"]]
        # keys have a few large channels, as attention keys do
        gain = 1.0 + 4.0 * (torch.rand((H, D), generator=gen, device=dev) > 0.95)
        st["k"] = (torch.randn((T, H, D), generator=gen, device=dev) * gain).to(dt)
        st["v"] = torch.randn((T, H, D), generator=gen, device=dev).to(dt)
        pages = -(-T // page) + 4
        # the tokens lie in pages handed out in no order
        order = torch.randperm(pages, generator=gen, device=dev)
        t = torch.arange(T, device=dev)
        st["slots"] = order[t // page] * page + t % page
        st["cache"] = _storage(pages, H, page, D, case["bits"], dt, dev)
        return st
    if case["op"] == "attention":
        H, D, page, bits = case["kv_heads"], case["dim"], case["page"], case["bits"]
        dt = DTYPES[case["dtype"]]
        lens = _lengths(case)
        need = [-(-length // page) for _, length in lens]
        pages, width = sum(need), max(need)
        order = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        first = [sum(need[:b]) for b in range(len(need))]
        rows = [torch.nn.functional.pad(order[f:f + n], (0, width - n)) for f, n in zip(first, need)]
        st["page_table"] = torch.stack(rows)
        st["kv_lens"] = torch.tensor([length for _, length in lens], dtype=torch.int32, device=dev)
        starts = [sum(n for n, _ in lens[:b]) for b in range(len(lens) + 1)]
        st["q_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        st["max_q_len"] = max(n for n, _ in lens)
        st["max_kv_len"] = max(length for _, length in lens)
        st["q"] = torch.randn((starts[-1], case["heads"], D), generator=gen, device=dev).mul_(1.5).to(dt)
        st["cache"] = c = _storage(pages, H, page, D, bits, dt, dev)
        st["scale"] = D ** -0.5
        for name in ("k", "v"):
            if bits == 16:
                c[name].normal_(generator=gen)
            elif bits == 8:
                c[name].copy_(torch.randint(-127, 128, c[name].shape, generator=gen, device=dev, dtype=torch.int8))
                c[name + "_scale"].uniform_(0.008, 0.02, generator=gen)
            else:
                c[name].copy_(torch.randint(0, 256, c[name].shape, generator=gen, device=dev, dtype=torch.uint8))
                c[name + "_scale"][..., 0].uniform_(0.15, 0.3, generator=gen)  # step
                c[name + "_scale"][..., 1] = c[name + "_scale"][..., 0] * -7.5  # value of code 0
                c[name + "_scale"][..., 1] += torch.randn(c[name + "_scale"].shape[:-1], generator=gen, device=dev) * 0.1
        return st
    B, n, V = case["seqs"], case["drafts"], case["vocab"]
    # a target whose likeliest tokens stand out, and a draft that mostly agrees with it
    logits = torch.randn((B, n + 1, V), generator=gen, device=dev) * 3.0
    draft = logits[:, :n] + torch.randn((B, n, V), generator=gen, device=dev) * 0.7
    q = torch.softmax(draft, -1)
    race = torch.empty((B, n, V), device=dev).exponential_(generator=gen)
    st["draft_tokens"] = (q / race).argmax(-1) if case["probs"] else draft.argmax(-1)
    st["draft_probs"] = q.to(DTYPES[case["probs"]]) if case["probs"] else None
    st["target_logits"] = logits.to(DTYPES[case["dtype"]])
    st["uniforms"] = torch.rand((B, n), generator=gen, device=dev)
    st["noise"] = torch.empty((B, V), device=dev).exponential_(generator=gen)
    st["draft_lens"] = torch.tensor(_draft_lengths(case), dtype=torch.int32, device=dev) if case["ragged"] else None
    st["temperature"] = None
    if case["temps"] == "mixed":
        t = torch.rand((B,), generator=gen, device=dev) + 0.3
        st["temperature"] = torch.where(torch.arange(B, device=dev) % 3 == 0, torch.zeros_like(t), t)
    return st


def _storage(pages, heads, page, dim, bits, dtype, dev):
    """A cache's tensors: [pages, heads, page, dim] 16-bit values, int8 codes with a float32
    scale a row, or 4-bit codes two to a byte (the even element in the low half) with a
    float32 (step, value of code 0) a row."""
    c = {"bits": bits, "dtype": dtype}
    for name in ("k", "v"):
        if bits == 16:
            c[name] = torch.zeros((pages, heads, page, dim), dtype=dtype, device=dev)
        elif bits == 8:
            c[name] = torch.zeros((pages, heads, page, dim), dtype=torch.int8, device=dev)
            c[name + "_scale"] = torch.zeros((pages, heads, page), device=dev)
        else:
            c[name] = torch.zeros((pages, heads, page, dim // 2), dtype=torch.uint8, device=dev)
            c[name + "_scale"] = torch.zeros((pages, heads, page, 2), device=dev)
    return c


# ------------------------------------------------------------------ one pass
def run(st):
    op = st["case"]["op"]
    if own:
        return _run_own(st)
    return {"cache": _plain_cache, "attention": _plain_attention, "verify": _plain_verify}[op](st)


def _run_own(st):
    from robustgemq_b200 import serving

    case = st["case"]
    if case["op"] == "verify":
        r = serving.verify_draft(st["target_logits"], st["draft_tokens"], st["uniforms"], st["noise"],
                                 draft_probs=st["draft_probs"], draft_lens=st["draft_lens"],
                                 temperature=st["temperature"])
        return {"tokens": r.tokens, "num_accepted": r.num_accepted, "logprobs": r.logprobs}
    c = st["cache"]
    cache = serving.PagedKVCache.from_tensors(c["k"], c["v"], c.get("k_scale"), c.get("v_scale"), dtype=c["dtype"])
    if case["op"] == "cache":
        cache.write(st["k"], st["v"], st["slots"])
        k, v = cache.read(st["slots"])
        return {"k": k, "v": v}
    r = serving.paged_attention(st["q"], cache, st["page_table"], st["kv_lens"], q_starts=st["q_starts"],
                                max_q_len=st["max_q_len"], max_kv_len=st["max_kv_len"], scale=st["scale"],
                                window=case["window"], return_lse=case["lse"])
    return {"out": r[0], "lse": r[1]} if case["lse"] else {"out": r}


def _plain_quantise(x, bits):
    x = x.float()
    if bits == 16:
        return x, None
    if bits == 8:
        most = x.abs().amax(-1).clamp_min(127 * MIN_SCALE)
        return torch.round(x * 127.0 / most[..., None]).clamp(-127, 127).to(torch.int8), most / 127.0
    lo = x.amin(-1)
    span = (x.amax(-1) - lo).clamp_min(15 * MIN_SCALE)
    q = torch.round((x - lo[..., None]) * 15.0 / span[..., None]).clamp(0, 15).to(torch.uint8)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.stack([span / 15.0, lo], -1)


def _plain_values(codes, scale, bits):
    if bits == 16:
        return codes.float()
    if bits == 8:
        return codes.float() * scale[..., None]
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return q * scale[..., :1] + scale[..., 1:]


def _plain_cache(st):
    c, bits = st["cache"], st["case"]["bits"]
    page = c["k"].shape[2]
    p, o = st["slots"] // page, st["slots"] % page
    out = {}
    for name in ("k", "v"):
        codes, scale = _plain_quantise(st[name], bits)
        c[name][p, :, o] = codes.to(c[name].dtype)
        if bits != 16:
            c[name + "_scale"][p, :, o] = scale
        got = c[name][p, :, o]
        out[name] = _plain_values(got, c[name + "_scale"][p, :, o] if bits != 16 else None, bits).to(c["dtype"])
    return out


def _plain_attention(st):
    case, c, q = st["case"], st["cache"], st["q"]
    bits, g = case["bits"], case["heads"] // case["kv_heads"]
    table = st["page_table"].long()
    kv_lens, starts = st["kv_lens"].long(), st["q_starts"].long()
    q_lens = starts[1:] - starts[:-1]
    B, T, n = table.shape[0], q.shape[0], st["max_q_len"]
    vals = []
    for name in ("k", "v"):
        x = _plain_values(c[name][table], c[name + "_scale"][table] if bits != 16 else None, bits)
        vals.append(x.transpose(1, 2).flatten(2, 3))  # [B, kv_heads, positions, dim]
    L = vals[0].shape[2]
    # the sequences' new tokens, padded to the longest
    i = torch.arange(n, device=q.device)
    qp = q[(starts[:-1, None] + i).clamp_max(T - 1)].float()  # [B, n, heads, dim]
    qp = qp.unflatten(2, (case["kv_heads"], g)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, kv_heads, g * n, dim]
    s = torch.matmul(qp, vals[0].transpose(2, 3)).mul_(st["scale"]).unflatten(2, (g, n))  # [B, kv_heads, g, n, L]
    pos = (kv_lens - q_lens)[:, None] + i  # [B, n]
    j = torch.arange(L, device=q.device)
    seen = (j <= pos[..., None]) & (j < kv_lens[:, None, None])
    if case["window"]:
        seen &= j > pos[..., None] - case["window"]
    s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    s.sub_(m).exp_()
    z = s.sum(-1, keepdim=True)
    o = torch.matmul(s.flatten(2, 3), vals[1]).unflatten(2, (g, n)) / torch.where(z == 0, 1.0, z)
    lse = (m + z.log()).squeeze(-1)
    # back to the packed tokens
    tok = torch.arange(T, device=q.device)
    b = torch.searchsorted(starts[1:], tok, right=True)
    at = tok - starts[b]
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[b, at].to(q.dtype)
    if not case["lse"]:
        return {"out": out}
    return {"out": out, "lse": lse.permute(0, 3, 1, 2).flatten(2, 3)[b, at]}


def _plain_verify(st):
    l, x = st["target_logits"].float(), st["draft_tokens"]
    B, n = x.shape
    V = l.shape[-1]
    temp = st["temperature"] if st["temperature"] is not None else torch.ones(B, device=l.device)
    l = l / torch.where(temp == 0, 1.0, temp)[:, None, None]
    first = l.argmax(-1, keepdim=True)
    l = l - l.amax(-1, keepdim=True)
    e = l.exp()
    z = e.sum(-1, keepdim=True)
    j = torch.arange(V, device=l.device)
    p = torch.where((temp == 0)[:, None, None], (j == first).float(), e / z)
    px = p[:, :n].gather(-1, x[..., None]).squeeze(-1)
    if st["draft_probs"] is not None:
        qx = st["draft_probs"].gather(-1, x[..., None]).squeeze(-1).float()
    else:
        qx = torch.ones_like(px)
    i = torch.arange(n + 1, device=l.device)
    lens = st["draft_lens"].long() if st["draft_lens"] is not None else torch.full((B,), n, device=l.device)
    ok = (st["uniforms"] * qx < px) & (i[:n] < lens[:, None])
    taken = ok.long().cumprod(-1).sum(-1)  # [B]
    b = torch.arange(B, device=l.device)
    pn = p[b, taken]
    at = taken.clamp_max(n - 1)
    qn = st["draft_probs"][b, at].float() if st["draft_probs"] is not None else (j == x[b, at][:, None]).float()
    left = torch.where((taken < lens)[:, None], (pn - qn).clamp_min(0), pn)
    left = torch.where(left.amax(-1, keepdim=True) > 0, left, pn)
    last = (left / st["noise"]).argmax(-1)
    xs = torch.nn.functional.pad(x, (0, 1))
    tokens = torch.where(i < taken[:, None], xs, torch.where(i == taken[:, None], last[:, None], -1))
    lp = (l - z.log()).gather(-1, tokens.clamp_min(0)[..., None]).squeeze(-1)
    return {"tokens": tokens, "num_accepted": taken.int(), "logprobs": torch.where(tokens >= 0, lp, 0.0)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"cache": _exact_cache, "attention": _exact_attention, "verify": _exact_verify}[case["op"]](st)


def _exact_cache(st):
    bits, out = st["case"]["bits"], {}
    for name in ("k", "v"):
        x = st[name].double()
        if bits == 8:
            most = torch.clamp(x.abs().max(-1, keepdim=True).values, min=127 * MIN_SCALE)
            x = torch.round(127 * x / most) * (most / 127)
        elif bits == 4:
            lo, hi = torch.aminmax(x, dim=-1, keepdim=True)
            span = torch.clamp(hi - lo, min=15 * MIN_SCALE)
            x = torch.round(15 * (x - lo) / span) * (span / 15) + lo
        out[name] = x
    return out


def _exact_rows(c, name, pages, head, length):
    """One sequence's keys or values of one head, [length, dim]."""
    raw = c[name][pages, head].flatten(0, 1)[:length]
    if c["bits"] == 16:
        return raw.double()
    sc = c[name + "_scale"][pages, head].flatten(0, 1)[:length].double()
    if c["bits"] == 8:
        return raw.double() * sc[:, None]
    both = torch.empty((raw.shape[0], 2 * raw.shape[1]), dtype=torch.float64, device=raw.device)
    both[:, 0::2] = (raw % 16).double()
    both[:, 1::2] = (raw // 16).double()
    return both * sc[:, 0:1] + sc[:, 1:2]


def _exact_attention(st):
    case, c = st["case"], st["cache"]
    g = case["heads"] // case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for b, (n, length) in enumerate(_lengths(case)):
        pages = st["page_table"][b, :-(-length // case["page"])].long()
        key = torch.arange(length, device="cuda")[None]
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        hide = key > pos
        if case["window"]:
            hide = hide | (key <= pos - case["window"])
        for h in range(case["kv_heads"]):
            k = _exact_rows(c, "k", pages, h, length)
            v = _exact_rows(c, "v", pages, h, length)
            for a in range(h * g, (h + 1) * g):
                s = (st["q"][at:at + n, a].double() @ k.T) * st["scale"]
                s = s.masked_fill(hide, -math.inf)
                row = torch.logsumexp(s, -1)
                out[at:at + n, a] = torch.exp(s - row[:, None]) @ v
                lse[at:at + n, a] = row
        at += n
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}


def _exact_verify(st):
    case = st["case"]
    B, n, V = case["seqs"], case["drafts"], case["vocab"]
    lens = _draft_lengths(case)
    lp = torch.zeros((B, n + 1), dtype=torch.float64, device="cuda")
    for b in range(B):
        t = 1.0 if st["temperature"] is None else float(st["temperature"][b])
        logs = torch.log_softmax(st["target_logits"][b].double() / (t or 1.0), -1)
        best = st["target_logits"][b].argmax(-1)
        for i in range(n + 1):
            p = logs[i].exp()
            if t == 0:
                p = torch.zeros_like(p)
                p[best[i]] = 1.0
            q = torch.zeros_like(p)
            if i < lens[b]:
                x = int(st["draft_tokens"][b, i])
                if st["draft_probs"] is not None:
                    q = st["draft_probs"][b, i].double()
                else:
                    q[x] = 1.0
                if float(st["uniforms"][b, i].double() * q[x]) < float(p[x]):
                    lp[b, i] = logs[i, x]
                    continue
            rest = torch.clamp(p - q, min=0)
            rest = rest if bool((rest > 0).any()) else p
            lp[b, i] = logs[i, int((rest / st["noise"][b].double()).argmax())]
            break
    return {"tokens": None, "num_accepted": None, "logprobs": lp}
