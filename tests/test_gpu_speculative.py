"""Several sequences decoded together on the paged cache with drafted tokens
(``inference/speculative.py``) against the same model's plain forward."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from robustgemq_b200.inference.generate import synthetic_olmoe

    return synthetic_olmoe(num_layers=2, seed=4, max_position_embeddings=1024)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("bits,bound", [(16, 5e-3), (8, 2e-2), (4, 3e-1)])
def test_chunks_on_the_paged_cache_match_the_model(model, bits, bound):
    """Two prompts in uneven chunks, side by side, against the model on each prompt whole.
    16 bits: the bound of the other fused-attention test (another order of sums). 8 and 4
    bits: keys and values move by half a step of max|x| / 127, or of the range / 15, about
    1% and 10% of their size, and so, at most, do a layer's attention outputs."""
    from robustgemq_b200 import _lib
    from robustgemq_b200.inference.speculative import PagedDecoder

    g = torch.Generator().manual_seed(1)
    a, b = (torch.randint(0, 50304, (n,), generator=g) for n in (150, 77))
    dec = PagedDecoder(model, num_pages=20, page_size=16, bits=bits)
    sa, sb = dec.add_sequence(), dec.add_sequence()
    rows = {sa: [], sb: []}
    for ca, cb in ((100, 1), (3, 60), (47, 16)):
        ta = a[dec.lengths[sa]:dec.lengths[sa] + ca].tolist()
        tb = b[dec.lengths[sb]:dec.lengths[sb] + cb].tolist()
        out = dec.forward([sa, sb], [ta, tb])
        rows[sa].append(out[:ca])
        rows[sb].append(out[ca:])
        dec.advance(sa, ca)
        dec.advance(sb, cb)
    with torch.no_grad():
        for s, ids in ((sa, a), (sb, b)):
            want = model(input_ids=ids.cuda()[None]).logits[0]
            assert _rel(torch.cat(rows[s]), want) <= bound
    assert _lib.device_error() == 0


@pytest.mark.parametrize("bits", [16, 8])
def test_greedy_generation_takes_the_models_tokens(model, bits):
    """Prompts that repeat themselves, so that lookups find drafts: every token that comes
    out has, in the plain forward of the whole text, a logit within the numerics' reach of
    the largest one there; drafts that are taken save steps."""
    from robustgemq_b200.inference.speculative import PagedDecoder

    g = torch.Generator().manual_seed(2)
    base = torch.randint(0, 50304, (40,), generator=g).tolist()
    prompts = [base + base, base[:7], base[::-1] + base[:20]]
    dec = PagedDecoder(model, num_pages=40, page_size=16, bits=bits)
    new, stats = dec.generate(prompts, max_new_tokens=24, drafts=3)
    assert [len(t) for t in new] == [24, 24, 24]
    assert 8 <= stats["steps"] <= 23 and stats["accepted"] <= stats["drafted"]
    assert len(dec.free) == 40  # every page given back
    with torch.no_grad():
        for p, t in zip(prompts, new):
            logits = model(input_ids=torch.tensor(p + t, device="cuda")[None]).logits[0].float()
            rows = logits[len(p) - 1:-1]
            got = rows[torch.arange(24), torch.tensor(t, device="cuda")]
            # 1% (16 bits) and 4% (8 bits) of the logits' spread: twice the bounds above
            assert (rows.amax(-1) - got <= (0.01 if bits == 16 else 0.04) * rows.std(-1) * 4).all()


def test_sampled_generation_is_reproducible(model):
    from robustgemq_b200.inference.speculative import PagedDecoder

    prompts = [[1, 2, 3, 1, 2, 3, 1, 2], [7] * 30]
    out = []
    for _ in range(2):
        dec = PagedDecoder(model, num_pages=16, page_size=32, bits=8)
        out.append(dec.generate(prompts, 12, drafts=4, temperature=0.8, generator=torch.Generator(device="cuda").manual_seed(5)))
    assert out[0] == out[1]


def test_a_full_cache_is_an_error(model):
    from robustgemq_b200.inference.speculative import PagedDecoder

    dec = PagedDecoder(model, num_pages=2, page_size=16)
    s = dec.add_sequence()
    dec.forward([s], [[1] * 32])
    dec.advance(s, 32)
    with pytest.raises(RuntimeError, match="full"):
        dec.forward([s], [[1]])
