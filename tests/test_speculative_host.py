"""``PagedDecoder``'s bookkeeping on the CPU: its checks, its pages and sequence numbers,
with the model's forward and the verification in place of the real ones."""

from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch
from torch import nn

VOCAB = 50


@pytest.fixture
def decoder(monkeypatch):
    """Eight pages of four tokens; every step's logits say "the token after the last one",
    and the verification takes no draft."""
    from robustgemq_b200.inference import speculative
    from robustgemq_b200.inference.generate import FusedOlmoeAttention

    class Attention(FusedOlmoeAttention):
        def __init__(self):
            nn.Module.__init__(self)
            self.head_dim = 16

    embed = nn.Embedding(VOCAB, 4)
    model = SimpleNamespace(
        model=SimpleNamespace(layers=[SimpleNamespace(self_attn=Attention())], embed_tokens=embed),
        config=SimpleNamespace(num_attention_heads=1, num_key_value_heads=1, vocab_size=VOCAB),
        parameters=embed.parameters)
    monkeypatch.setattr(speculative, "PagedKVCache", lambda *args, **kw: None)
    dec = speculative.PagedDecoder(model, num_pages=8, page_size=4)
    dec.seen = []

    def run(seqs, chunks):
        dec.seen.append([list(c) for c in chunks])
        for s, c in zip(seqs, chunks):
            dec._reserve(s, dec.lengths[s] + len(c))
        logits = torch.zeros((sum(map(len, chunks)), VOCAB))
        last = torch.tensor([t for c in chunks for t in c])
        logits[torch.arange(len(last)), (last + 1) % VOCAB] = 1.0
        return logits

    def verify(logits, drafts, uniforms, noise, draft_lens=None, temperature=None):
        tokens = torch.full((logits.shape[0], logits.shape[1]), -1)
        tokens[:, 0] = logits[:, 0].argmax(-1)
        return speculative.Verified(tokens, torch.zeros(logits.shape[0], dtype=torch.int32), torch.zeros(tokens.shape))

    monkeypatch.setattr(dec, "forward", run)
    monkeypatch.setattr(speculative, "verify_draft", verify)
    return dec


def test_generate_on_the_stand_ins(decoder):
    new, stats = decoder.generate([[1, 2], [7]], 4)
    assert new == [[3, 4, 5, 6], [8, 9, 10, 11]] and stats["steps"] == 3
    assert sorted(decoder.free) == list(range(8))


@pytest.mark.parametrize("after", [0, 2])
def test_a_row_without_a_distribution_ends_generation(decoder, monkeypatch, after):
    """The verification's -1 is an error, and no step is given it as a token."""
    from robustgemq_b200.inference import speculative

    whole, calls = speculative.verify_draft, []

    def verify(*args, **kw):
        calls.append(1)
        r = whole(*args, **kw)
        if len(calls) > after:
            r.tokens[-1] = -1
        return r

    monkeypatch.setattr(speculative, "verify_draft", verify)
    with pytest.raises(RuntimeError, match="distribution"):
        decoder.generate([[1, 2], [7]], 6)
    assert all(0 <= t < VOCAB for chunks in decoder.seen for c in chunks for t in c)


@pytest.mark.parametrize("temperature", [-1.0, math.nan, math.inf])
def test_temperatures_that_are_none(decoder, temperature):
    with pytest.raises(ValueError, match="temperature"):
        decoder.generate([[1, 2]], 2, temperature=temperature)
    assert decoder.seen == []


@pytest.mark.parametrize("token", [-1, VOCAB, 1 << 40])
def test_tokens_outside_the_vocabulary_do_not_reach_the_model(decoder, monkeypatch, token):
    """An index outside the embedding is a fault on the device, so the host looks."""
    monkeypatch.undo()  # the decoder's own forward
    s = decoder.add_sequence()
    with pytest.raises(ValueError, match="vocabulary"):
        decoder.forward([s], [[1, token, 2]])
    assert decoder.pages[s] == []


def test_pages_come_back_after_an_error(decoder):
    with pytest.raises(RuntimeError, match="full"):
        decoder.generate([[1] * 12, [2] * 12, [3] * 12], 4)
    assert sorted(decoder.free) == list(range(8))
    new, _ = decoder.generate([[1, 2, 3]], 3)
    assert new == [[4, 5, 6]]


def test_pages_come_back_after_a_step_that_failed(decoder, monkeypatch):
    whole = decoder.forward

    def run(seqs, chunks):
        if len(decoder.seen) == 3:
            raise KeyError("no")
        return whole(seqs, chunks)

    monkeypatch.setattr(decoder, "forward", run)
    with pytest.raises(KeyError):
        decoder.generate([[1, 2], [3]], 5)
    assert sorted(decoder.free) == list(range(8)) and decoder.lengths == [0, 0]


def test_released_numbers_are_given_out_again(decoder):
    """Many calls on one decoder do not grow its tables."""
    for _ in range(5):
        decoder.generate([[1, 2], [3], [4]], 3)
    assert decoder.page_table.shape[0] == len(decoder.pages) == len(decoder.lengths) == 3
    a = decoder.add_sequence()
    b = decoder.add_sequence()
    decoder.release(a)
    decoder.release(a)
    c, d = decoder.add_sequence(), decoder.add_sequence()
    assert c == a and len({b, c, d}) == 3


def test_nothing_to_generate(decoder):
    none = {"steps": 0, "drafted": 0, "accepted": 0}
    assert decoder.generate([[1, 2], [3]], 0) == ([[], []], none)
    assert decoder.generate([], 5) == ([], none)
    assert decoder.seen == [] and decoder.generate([[1]], 1)[0] == [[2]]


@pytest.mark.parametrize("args,text", [
    (dict(prompts=[[1], []]), "prompt"), (dict(max_new_tokens=-1), "max_new_tokens"), (dict(drafts=-1), "drafts"),
    (dict(chunk=0), "chunk"),
])
def test_generate_refusals(decoder, args, text):
    with pytest.raises(ValueError, match=text):
        decoder.generate(**(dict(prompts=[[1, 2]], max_new_tokens=3) | args))
    assert decoder.seen == [] and sorted(decoder.free) == list(range(8))


@pytest.mark.parametrize("seqs", [[0, 0], [0, 2], [-1, 0]])
def test_forward_takes_a_sequence_once(decoder, monkeypatch, seqs):
    """Two chunks of one sequence would be written to the same places."""
    monkeypatch.undo()
    decoder.add_sequence(), decoder.add_sequence()
    with pytest.raises(ValueError, match="once a call"):
        decoder.forward(seqs, [[1, 2], [3]])
    assert decoder.pages == [[], []]
